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
  int words;     // where a row's words begin
  float* states;  // max and sum of each of part's slots and heads
  int32_t* range;  // [tokens][2]: the first and the last share that has units of the token (of those with keys)
};

// ---------------------------------------------------------------------------
// Any head size, block size and head group, as attn_any_kernel: a workgroup is GH query heads of one (token, kv
// head), its 4 waves take the chunks in turn; a lane is a key in the scores and head dimensions lane + 64 i in P . V;
// fp32 math.
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
  for (int c = w; c < (L + kChunk - 1) / kChunk; c += kGenWaves) {
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
// Codes as fp16: a nibble at bits 0 .. 3 of a half word, or'ed with 0x6400, is the number 1024 + n, at bits 4 .. 7
// with 0x5400 64 + n (their last places are 1 and 1/16).  Adding -(1024 + z) or -(64 + z) and multiplying by d are
// exact in fp16: n - z has four bits and a sign, d seven.
struct Kv4Half {  // a pair of groups' (or one group's, twice) scale and offsets
  f16x2 d, z_low, z_high;
};
// The magic numbers stay in registers: (x & mask) | magic is then one v_and_or_b32, which takes one scalar and no
// literal.
struct Kv4Magic {
  uint32_t low = 0x64006400u, high = 0x54005400u, mixed = 0x54006400u, z_low = 0xE400E400u, z_high = 0xD400D400u;
  __device__ __forceinline__ Kv4Magic() {
    asm volatile("" : "+v"(low), "+v"(high), "+v"(mixed), "+v"(z_low), "+v"(z_high));
  }
  // words: a word in each half
  __device__ __forceinline__ Kv4Half half(uint32_t words) const {
    return {__builtin_bit_cast(f16x2, words & 0xFFF0FFF0u), __builtin_bit_cast(f16x2, (words & 0x000F000Fu) | z_low),
            __builtin_bit_cast(f16x2, (words << 4 & 0x00F000F0u) | z_high)};
  }
  // the nibbles of x at bits 0 .. 3 and 16 .. 19, and those at 4 .. 7 and 20 .. 23, as values
  __device__ __forceinline__ uint32_t lows(uint32_t x, const Kv4Half& h) const {
    return __builtin_bit_cast(uint32_t, (__builtin_bit_cast(f16x2, (x & 0x000F000Fu) | low) + h.z_low) * h.d);
  }
  __device__ __forceinline__ uint32_t highs(uint32_t x, const Kv4Half& h) const {
    return __builtin_bit_cast(uint32_t, (__builtin_bit_cast(f16x2, (x & 0x00F000F0u) | high) + h.z_high) * h.d);
  }
  // eight dimensions (a dword of codes) in the order 0 4 1 5 2 6 3 7
  __device__ __forceinline__ u32x4 eight(uint32_t codes, const Kv4Half& h) const {
    const uint32_t up = codes >> 8;
    return u32x4{lows(codes, h), highs(codes, h), lows(up, h), highs(up, h)};
  }
};

// A row of q as operands of the fp16 matrix cores: times 2^shift, so that its largest value lies in [2^10, 2^11),
// which fp16 holds to 2^-24 beside it.  q of 16 bits is exact so down to 2^-24 of the largest, and below within 2^-35
// of it; fp32 takes two operands, what is left of each value in the second.
template <typename T>
constexpr int kQParts = sizeof(T) == 4 ? 2 : 1;
__device__ __forceinline__ int q_shift(float largest) {
  const int e = (int)(__builtin_bit_cast(uint32_t, largest) >> 23);  // biased; subnormal ones stay small
  return e == 0 || e == 255 ? 0 : 137 - e;
}
// What such a row's scores are multiplied by, in exp2 units.  Above zero, so that masked scores stay -inf, and
// finite, so that zeros stay zeros: past either end the weights are equal, or fp32 scores are infinite.
__device__ __forceinline__ float q_scale(float scale_log2, int shift) {
  return fminf(fmaxf(ldexpf(scale_log2, -shift), 0x1p-126f), 0x1.fffffep127f);
}

// The lead that the weights' fp16 numbers need (attention_tiles.hpp): the far one where the output is fp32 and shows
// it.  It costs the rescalings: 16-bit types take the near one, with which 256 ragged sequences take 152 us, with the
// far one 154.
template <typename T>
constexpr float kKv4Lazy = sizeof(T) == 4 ? kFarLazy : kLazyMax;
template <typename T>
constexpr float kKv4Lead = sizeof(T) == 4 ? kFarLead : kLead;
using Kv4Mma = AttnMma<_Float16>;
typedef Kv4Mma::v8 h8;
typedef unsigned short us2 __attribute__((ext_vector_type(2)));

// One token: a wave is (token, kv head, 16 of its heads) and takes 32 keys at a time on its own:
//   S^T = K . Q^T     16x16x32 MFMAs: lane (row of 16 keys, quarter of the head) loads its codes in one go and
//                     turns them into the operand, one scale a lane (head size 256: two)
//   O^T += V^T . P^T  a lane holds head dimensions HD / 16 r .. of eight keys; byte b of two keys' codes side by side
//                     (one v_perm) is the low nibbles' operand of tile 2 b and the high ones' of 2 b + 1, so V needs no
//                     transpose; B = S^T's registers, P in two parts
// A workgroup's waves take HEADS kv heads side by side, so that each row's bytes are read together, and share out the
// keys where the heads are few.  A unit's rows (those heads' codes and words) come to LDS by DMA, one unit ahead of
// the waves, which take theirs into registers at once: straight from memory a wave would read 64 bytes of each line,
// four waves one after the other, from caches that do not hold what all of a CU's waves have in flight (256 sequences
// of 4096 keys 171 us with three workgroups a CU, 150 with two).
// Bound by vector instructions, 364 for a wave's 32 keys (59% of issue cycles; the MFMAs 16%), beside HBM: 256 ragged
// sequences of up to 8192 keys, 28 / 4 heads of 128, bf16, 150 us, 4.1 TB/s of codes and words, where a copy's rate
// gives 94.
template <int HD, int HEADS>
struct Kv4Lds {
  static constexpr int kWaves = HEADS > 4 ? HEADS : 4, kWays = kWaves / HEADS;
  // 16-byte units of a row
  static constexpr int kCodes = HEADS * HD / 32, kWords = HEADS * HD >= 256 ? HEADS * HD / 256 : 1;
  static constexpr int kRow = 16 * (kCodes + kWords), kSlab = 16 * kRow, kUnit = 4 * kSlab;  // K, K, V, V
  static constexpr int kBuf = kWays * kUnit;
  static constexpr int kState = HD * 16 + 32;  // O^T [HD][16], m [16], l [16] of a wave
  static constexpr int kStates = kWays > 1 ? kWaves * kState * (int)sizeof(float) : 0;
  static constexpr int kBytes = 2 * kBuf > kStates ? 2 * kBuf : kStates;
};

// The softmax state of one (token, head) over every step-th run of `keys` keys (at most 64) from run c0 to c1, by one
// wave without the matrix cores: for rows whose result is not finite, since 0 * V of a masked key that is no number
// would reach them there.  Lane = key, then dimensions lane + 64 i.
template <int DPL, typename T>
__device__ __forceinline__ void kv4_row_state(const Kv4Args<T>& a, int c0, int c1, int step, int keys, int seq,
                                              int64_t t, int h, int kvh, int L, float& m, float& l,
                                              float (&acc)[DPL]) {
  const int lane = threadIdx.x & 63, words = a.words + kvh * (a.hd / 16), codes = kvh * (a.hd / 2);
  const T* q = a.q + t * a.q_stride + (int64_t)h * a.hd;
  m = -INFINITY;
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < DPL; ++i) acc[i] = 0.0f;
#pragma unroll 1
  for (int c = c0; c < c1; c += step) {
    const int key = c * keys + lane;
    const bool seen = lane < keys && key < L;
    const int block = seen ? key_block(a, seq, key) : -1;
    const int64_t row = block >= 0 ? (int64_t)block * a.bs + key % a.bs : 0;
    float s = block >= 0 ? 0.0f : __builtin_nanf("");
    if (block >= 0) {
      const uint8_t* kp = a.k + row * a.row_bytes;
#pragma unroll 1
      for (int d = 0; d < a.hd; ++d) {
        const uint32_t word = *reinterpret_cast<const uint16_t*>(kp + words + 2 * (d / kKv4Group));
        s = fmaf(to_f32(q[d]), kv4_value(word, (uint32_t)kp[codes + d / 2] >> (4 * (d & 1)) & 15u), s);
      }
    }
    const float x = seen ? s * a.scale_log2 : -INFINITY;
    const float m_new = fmaxf(m, wave_max(x)), m_use = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m - m_use), p = __builtin_amdgcn_exp2f(x - m_use);
    l = l * alpha + wave_sum(p);
    m = m_new;
#pragma unroll
    for (int i = 0; i < DPL; ++i) acc[i] *= alpha;
    for (uint64_t left = __ballot(seen); left; left &= left - 1) {
      const int j = __builtin_ctzll(left);
      const float pj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, p), j));
      const int64_t rj = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)row, j) |
                         (int64_t)__builtin_amdgcn_readlane((int)(row >> 32), j) << 32;
      const uint8_t* vp = a.v + rj * a.row_bytes;
#pragma unroll
      for (int i = 0; i < DPL; ++i) {
        const int d = lane + 64 * i;
        if (d < a.hd)
          acc[i] = fmaf(pj, kv4_value(*reinterpret_cast<const uint16_t*>(vp + words + 2 * (d / kKv4Group)),
                                      (uint32_t)vp[codes + d / 2] >> (4 * (d & 1)) & 15u), acc[i]);
      }
    }
  }
}

// What a workgroup does for n tokens of one sequence from t on, whose heads fill the 16 columns (or for one of more
// heads): units [u0, u1) of their keys, of which the token that sees most sees L; their states go to part's slots
// from `slot` on unless that is all of them.
struct Kv4Job {
  int64_t t, slot;
  int n, L, u0, u1;
};

// GROUPS: several tokens may fill the columns.  (Single tokens without it keep their keys' count in a scalar: with it
// 256 ragged sequences take 162 us instead of 148.)
template <typename T, int HD, int HEADS, bool GROUPS>
__device__ __forceinline__ void kv4_attend_token(const Kv4Args<T>& a, const FastDiv& div, const Kv4Job& job, int rest,
                                                 uint8_t* lds) {
  using Lds = Kv4Lds<HD, HEADS>;
  constexpr int kWays = Lds::kWays;             // waves that share a head's keys
  constexpr int kTiles = HD / 16, kSteps = HD / 32;
  constexpr int kKDwords = HD / 32;             // codes of a lane in K: HD / 4 dimensions
  constexpr int kKGroups = HD > 128 ? HD / 128 : 1;
  constexpr int kVBytes = HD / 32;              // of a lane in V: HD / 16 dimensions
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int col = lane & 15, g = lane >> 4;
  const int G = a.q_heads / a.kv_heads, parts = (G + 15) / 16;
  const int kvh0 = rest / parts * HEADS, side = wave % HEADS, kvh = kvh0 + side;
  const int part = rest % parts, way = wave / HEADS;
  const int i0 = GROUPS && job.n > 1 ? col / G : 0;  // this column's token and head
  const int64_t t = job.t + i0;
  const int h = kvh * G + 16 * part + col - i0 * G;
  const bool ok = i0 < job.n && h < (kvh + 1) * G;
  const int L = job.L, seq = __builtin_amdgcn_readfirstlane(a.qseq[job.t]);
  const int own = !GROUPS ? L : ok ? key_count(a, t) : 0;  // the column's keys
  const int all = !GROUPS ? L : __builtin_amdgcn_readfirstlane(-wave_max_int(ok ? -own : -INT32_MAX));  // what all see
  const uint32_t row_b = (uint32_t)a.row_bytes;

  // q: operand element j of step s is dimension HD / 4 g + 8 s + {0, 4, 1, 5, 2, 6, 3, 7}[j]
  h8 qf[kQParts<T>][kSteps];
  float to_exp2;
  {
    float x[kSteps][8], most = 0.0f;
    const T* q = a.q + t * a.q_stride + (int64_t)h * HD + HD / 4 * g;
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int e = 0; e < 8; e += Pack<T>::N) {
        if (ok) Pack<T>::unpack(ld16(q + 8 * s + e), x[s] + e);
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
    to_exp2 = q_scale(a.scale_log2, shift);
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

  // The transfers.  A way's unit is four slabs' pieces, K and V of its first and last 16 keys, and its HEADS waves
  // take 4 / HEADS of them each (eight waves: half a piece); 16-byte unit i of a piece is row i / kRow's.
  const Kv4Slabs table(a, div, seq, L);
  constexpr int kRowUnits = Lds::kRow / 16, kHalves = HEADS > 4 ? HEADS / 4 : 1, kPieces = HEADS > 4 ? 1 : 4 / HEADS;
  constexpr int kPerWave = 16 * kRowUnits / kHalves, kTransfers = (kPerWave + 63) / 64;
  const uint32_t code0 = (uint32_t)(kvh0 * (HD / 2)), word0 = (uint32_t)(a.words + kvh0 * (HD / 16));
  const int part0 = HEADS > 4 ? side / 4 * kPerWave : 0;  // the wave's first 16-byte unit of its piece
  uint32_t from[kTransfers];
#pragma unroll
  for (int i = 0; i < kTransfers; ++i) {
    const int x = part0 + 64 * i + lane, r = x / kRowUnits, p = x - r * kRowUnits;
    from[i] = (uint32_t)r * row_b + (p < Lds::kCodes ? code0 + 16 * p : (word0 & ~15u) + 16 * (p - Lds::kCodes));
  }
  const auto piece_of = [&](int i) { return HEADS > 4 ? side & 3 : kPieces * side + i; };  // K, K, V, V
  SlabEntry e[kPieces];  // of the unit to load next
  const auto entries = [&](int u) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) e[i] = table.entry(32 * u + 16 * (piece_of(i) & 1));
  };
  const auto fetch = [&](int buf) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int piece = piece_of(i);
      uint8_t* dst = lds + buf * Lds::kBuf + way * Lds::kUnit + piece * Lds::kSlab + 16 * part0;
      if (piece < 2 && table.bad(e[i])) {  // keys without a block: no numbers, so NaN where they are seen
        for (int x = lane; x < kPerWave; x += 64) st16(dst + 16 * x, u32x4{~0u, ~0u, ~0u, ~0u});
        continue;
      }
      const __amdgpu_buffer_rsrc_t r = rows_rsrc((piece < 2 ? a.k : a.v) + table.at(e[i]), table.bytes(e[i]));
#pragma unroll
      for (int x = 0; x < kTransfers; ++x)
        if (64 * x + 64 <= kPerWave || 64 * x + lane < kPerWave) dma16(r, dst + 1024 * x, from[x]);
    }
  };
  // Where a lane finds its own: row col (K) or 4 g + i (V) of a slab.
  const uint32_t word = Lds::kCodes * 16 + (word0 & 15u) + side * (HD / 16);
  const uint32_t k_at = (uint32_t)col * Lds::kRow + side * (HD / 2) + HD / 8 * g;
  const uint32_t kw_at = (uint32_t)col * Lds::kRow + word + 2 * (HD / 4 * g / kKv4Group);
  const uint32_t v_at = (uint32_t)(4 * g) * Lds::kRow + side * (HD / 2) + kVBytes * col;
  const uint32_t vw_at = (uint32_t)(4 * g) * Lds::kRow + word + 2 * (HD / 16 * col / kKv4Group);
  const Kv4Magic magic;
  const int rounds = (job.u1 - job.u0 + kWays - 1) / kWays;
  if (rounds > 0) {
    entries(job.u0 + way);
    fetch(0);
    entries(job.u0 + way + kWays);
  }
#pragma unroll 1
  for (int round = 0; round < rounds; ++round) {
    const int u = job.u0 + round * kWays + way;
    tile_hand_over();  // this round's rows are in LDS, and every wave has the last one's in registers
    const uint8_t* unit = lds + (round & 1) * Lds::kBuf + way * Lds::kUnit;
    uint32_t kc[2][kKDwords], kw[2], vc[2][4][(kVBytes + 3) / 4];
    us2 vw[2][2];  // of two keys
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      const uint8_t* ks = unit + kt * Lds::kSlab;
      const uint8_t* vs = unit + (2 + kt) * Lds::kSlab;
      if constexpr (kKDwords == 2) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(ks + k_at);
        kc[kt][0] = w[0];
        kc[kt][1] = w[1];
      } else {
#pragma unroll
        for (int i = 0; i < kKDwords / 4; ++i) {
          const u32x4 w = ld16(ks + k_at + 16 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j) kc[kt][4 * i + j] = w[j];
        }
      }
      if constexpr (kKGroups == 2) kw[kt] = *reinterpret_cast<const uint32_t*>(ks + kw_at);
      else kw[kt] = *reinterpret_cast<const uint16_t*>(ks + kw_at);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* p = vs + v_at + i * Lds::kRow;
        if constexpr (kVBytes == 2) vc[kt][i][0] = *reinterpret_cast<const uint16_t*>(p);
        else if constexpr (kVBytes == 4) vc[kt][i][0] = *reinterpret_cast<const uint32_t*>(p);
        else {
          const u32x2 w = *reinterpret_cast<const u32x2*>(p);
          vc[kt][i][0] = w[0];
          vc[kt][i][1] = w[1];
        }
        vw[kt][i / 2][i % 2] = *reinterpret_cast<const uint16_t*>(vs + vw_at + i * Lds::kRow);
      }
    }
    __builtin_amdgcn_sched_barrier(0);  // (in front of LDS reads the compiler waits for transfers in flight: none is)
    if (round + 1 < rounds) {
      fetch((round & 1) ^ 1);
      entries(u + 2 * kWays);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (kWays > 1 && u >= job.u1) continue;
    f32x4 st[2];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      st[kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int gr = 0; gr < kKGroups; ++gr) {
        const uint32_t w = kKGroups == 1 ? kw[kt] : gr == 0 ? kw[kt] & 0xFFFFu : kw[kt] >> 16;
        const Kv4Half h = magic.half((w & 0xFFFFu) | w << 16);
#pragma unroll
        for (int i = 0; i < kSteps / kKGroups; ++i) {
          const int s = kSteps / kKGroups * gr + i;
          const h8 k = __builtin_bit_cast(h8, magic.eight(kc[kt][s], h));
#pragma unroll
          for (int p = 0; p < kQParts<T>; ++p) st[kt] = Kv4Mma::mma(k, qf[p][s], st[kt]);
        }
      }
    }
    // element j of tile kt is key 32 u + 16 kt + 4 g + j
    float mx = -INFINITY;
    if (32 * u + 32 > all) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (32 * u + 16 * kt + 4 * g + j >= own) st[kt][j] = -INFINITY;
    }
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int j = 0; j < 4; ++j) mx = fmaxf(mx, st[kt][j]);
    if (__any(fmaf(mx, to_exp2, -kKv4Lead<T>) > m + kKv4Lazy<T>)) {  // as in attend_token
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float m_new = fmaxf(m, fmaf(mx, to_exp2, -kKv4Lead<T>));
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
        pl[4 * kt + j] = (_Float16)fmaf((float)ph[4 * kt + j], -1.0f, p);
      }
    Kv4Half h[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) h[p] = magic.half(__builtin_bit_cast(uint32_t, vw[p / 2][p % 2]));
#pragma unroll
    for (int b = 0; b < kVBytes; ++b) {
      u32x4 low, high;
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const uint32_t pair = __builtin_amdgcn_perm(vc[p / 2][2 * (p % 2) + 1][b / 4], vc[p / 2][2 * (p % 2)][b / 4],
                                                    0x0C040C00u + 0x00010001u * (b % 4));
        low[p] = magic.lows(pair, h[p]);
        high[p] = magic.highs(pair, h[p]);
      }
      o[2 * b] = Kv4Mma::mma(__builtin_bit_cast(h8, low), ph, o[2 * b]);
      o[2 * b] = Kv4Mma::mma(__builtin_bit_cast(h8, low), pl, o[2 * b]);
      o[2 * b + 1] = Kv4Mma::mma(__builtin_bit_cast(h8, high), ph, o[2 * b + 1]);
      o[2 * b + 1] = Kv4Mma::mma(__builtin_bit_cast(h8, high), pl, o[2 * b + 1]);
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if constexpr (GROUPS) {  // columns that do not see all of the group's keys, and are not finite
    float finite = l * 0.0f;
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) finite = fmaf(o[j][i], 0.0f, finite);
    finite += __shfl_xor(finite, 16);
    finite += __shfl_xor(finite, 32);
#pragma unroll 1
    for (uint64_t left = __ballot(ok && own < L && !(finite == 0.0f)) & 0xFFFFu; left; left &= left - 1) {
      const int c = __builtin_ctzll(left);
      float mc, lc, acc[HD / 64];
      kv4_row_state<HD / 64>(a, job.u0 + way, job.u1, kWays, 32, seq, job.t + __builtin_amdgcn_readlane(i0, c),
                             __builtin_amdgcn_readlane(h, c), kvh, __builtin_amdgcn_readlane(own, c), mc, lc, acc);
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = kTiles * (4 * g + i) + j;
          float x = 0.0f;
#pragma unroll
          for (int k = 0; k < HD / 64; ++k) {
            const float y = __shfl(acc[k], d & 63);
            x = d >> 6 == k ? y : x;
          }
          o[j][i] = col == c ? x : o[j][i];
        }
      m = col == c ? mc : m;
      l = col == c ? lc : l;
    }
  }

  // O^T: lane column = head, element i of tile j dimension kTiles (4 g + i) + j
  if constexpr (kWays > 1) {
    float* state = reinterpret_cast<float*>(lds);
    __syncthreads();  // (a way's rows may still be read)
    float* own = state + wave * Lds::kState;
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
    for (int w = 0; w < kWays; ++w) mall = fmaxf(mall, state[(wave + w * HEADS) * Lds::kState + HD * 16 + col]);
    l = 0.0f;
#pragma unroll
    for (int j = 0; j < kTiles; ++j) o[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < kWays; ++w) {
      const float* of = state + (wave + w * HEADS) * Lds::kState;
      const float mw = of[HD * 16 + col], sc = mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mw - mall);
      l += sc * of[HD * 16 + 16 + col];  // (no keys: O = l = 0, or NaN)
#pragma unroll
      for (int j = 0; j < kTiles; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][i] += sc * of[(kTiles * (4 * g + i) + j) * 16 + col];
    }
    m = mall;
  }
  if (!ok) return;
  if (job.u0 > 0 || 32 * job.u1 < L) {
    const int64_t pi = (job.slot + i0) * a.q_heads + h;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < kTiles; j += 4)
        st16(a.part + pi * HD + kTiles * (4 * g + i) + j,
             __builtin_bit_cast(u32x4, f32x4{o[j][i], o[j + 1][i], o[j + 2][i], o[j + 3][i]}));
    if (g == 0) {
      float* ml = a.states + 2 * pi;
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
        *reinterpret_cast<t4*>(a.out + (t * a.q_heads + h) * HD + kTiles * (4 * g + i) + j) = v;
      }
  }
}

// The units of a batch's tokens, one group of tokens after the other, in equal shares: workgroups of a ragged batch
// end together.  A group is consecutive tokens of one sequence between two multiples of `group` (what a token's heads
// leave of the 16 columns), with the keys of the one that sees most.  Share w is units [w n, (w + 1) n) of the whole,
// which may end one group and begin others; its state of token t goes to slot w group + t, which no other pair has: a
// share's tokens follow those of the shares before, but for the one group (of at most `group` tokens) that both may
// have a part of.
// Every workgroup adds up the batch's units for that (a lane those of tokens / 64 tokens, at most 64 of them), which
// in the end costs more than equal shares gain.  In shares, and a workgroup each (for each group), over up to 4096
// and up to 1024 keys, bf16: 32 / 8 heads of 128, 2000 single tokens 989 and 1140, 315 and 324 us (14 / 2 heads of
// 64: 200 and 198, 81 and 61); 128 sequences of 5 tokens 225 and 395, 109 and 114; 128 of 8 282 and 390, 162 and 97
// (14 / 2, fp32: 152 and 94, 130 and 36).
constexpr int kShareTokens = 2048, kShareGroupTokens = 768;
constexpr int kLeastShare = 4;  // units
struct Kv4Group {
  int n, L, units;  // tokens (0: t does not begin a group), keys, units
};
template <bool GROUPS, typename T>
__device__ __forceinline__ Kv4Group kv4_group(const AttnArgs<T>& a, int64_t t, int group) {
  Kv4Group x{0, 0, 0};
  if constexpr (!GROUPS) {  // (no branch, so that a loop's loads go out together)
    const int L = key_count(a, min(t, a.tokens - 1));
    x.n = t < a.tokens;
    x.L = x.n ? L : 0;
  } else {
    if (t >= a.tokens) return x;
    const int at = (int)(t % group);
    const int32_t before = a.qseq[at > 0 ? t - 1 : t], seq = a.qseq[t];
    bool same = at == 0 || before != seq;
    for (int i = 0; i < group; i += 4) {  // four tokens' loads at once
      int32_t s[4];
      int L[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t y = min(t + i + k, a.tokens - 1);
        s[k] = a.qseq[y];
        L[k] = key_count(a, y);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        same = same && at + i + k < group && t + i + k < a.tokens && s[k] == seq;
        x.n += same;
        x.L = max(x.L, same ? L[k] : 0);
      }
    }
  }
  x.units = (x.L + 31) / 32;
  return x;
}
__device__ __forceinline__ int wave_prefix(int v) {  // the sum of this lane's and those below
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(v, d);
    if (lane >= d) v += up;
  }
  return v;
}
__device__ __forceinline__ int share_of(int64_t total, int shares) {
  return max((int)((total + shares - 1) / shares), kLeastShare);
}

// Waves of a SIMD: four, of 128 VGPRs, where that spills a little outside the loops; groups of a head size of 128
// three (16 sequences of 4 tokens 38 -> 31 us), but for workgroups of eight waves, of which three a SIMD hold one;
// two where q or O fill more registers (head size 256, or 128 in fp32: `q_dims`, of both of fp32's operands).
constexpr int kv4_waves_per_simd(int q_dims, int hd, int heads, bool groups) {
  return q_dims > 128 ? 2 : groups && hd == 128 && heads < 8 ? 3 : 4;
}
template <typename T, int HD, int HEADS, bool GROUPS>
__global__ __launch_bounds__((Kv4Lds<HD, HEADS>::kWaves * 64))
__attribute__((amdgpu_waves_per_eu(kv4_waves_per_simd(HD * kQParts<T>, HD, HEADS, GROUPS)))) void kv4_token_kernel(
    const Kv4Args<T> a, const FastDiv div, int shares, int group, int64_t first, int tile_tokens) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const int per_token = a.kv_heads / HEADS * ((a.q_heads / a.kv_heads + 15) / 16);
  const int w = (int)(blockIdx.x / per_token), rest = (int)(blockIdx.x % per_token);
  int64_t t = first + w;
  if (tile_tokens > 0) {  // tokens of tiles that kv4_tile_kernel leaves
    const int64_t t0 = t / tile_tokens * tile_tokens;
    const int n = a.tokens - t0 < tile_tokens ? (int)(a.tokens - t0) : tile_tokens;
    if (TileRuns(a.qseq, t0, n).count() <= kTileMaxRuns) return;
  }
  if (GROUPS && shares == 0) {  // the tokens at multiples of `group` first, which all begin groups: over all XCDs
    const int blocks = (int)((a.tokens + group - 1) / group);
    t = (int64_t)(w % blocks) * group + w / blocks;
    if (t >= a.tokens) return;
  }
  int u = 0, left = 0;
  if (shares > 0) {
    // the token in which the share begins: a lane's tokens first, then token by token
    const int per = (int)((a.tokens + 63) / 64);
    int sum = 0;
    for (int i = 0; i < per; ++i) sum += kv4_group<GROUPS>(a, (int64_t)lane * per + i, group).units;
    int up_to = wave_prefix(sum);
    const int total = __builtin_amdgcn_readlane(up_to, 63), share = share_of(total, shares);
    if ((int64_t)w * share >= total) return;
    const int begin = w * share;
    left = min(share, total - begin);
    const int from = __builtin_ctzll(__ballot(up_to > begin));
    const int before = __builtin_amdgcn_readlane(up_to - sum, from);
    const int own = lane < per ? kv4_group<GROUPS>(a, (int64_t)from * per + lane, group).units : 0;
    up_to = before + wave_prefix(own);
    const int at = __builtin_ctzll(__ballot(up_to > begin));
    t = (int64_t)from * per + at;
    u = begin - __builtin_amdgcn_readlane(up_to - own, at);
  }
#pragma unroll 1
  while (true) {
    const Kv4Group x = kv4_group<GROUPS>(a, t, group);
    const int tokens = __builtin_amdgcn_readfirstlane(x.n), L = __builtin_amdgcn_readfirstlane(x.L);
    const int units = (L + 31) / 32;
    const int n = shares > 0 ? min(units - u, left) : units;  // (no shares: the whole of a group, with keys or not)
    if (shares > 0 && n > 0 && rest == 0 && (int)threadIdx.x < tokens) {
      int32_t* range = a.range + 2 * (t + threadIdx.x);
      if (u == 0) range[0] = w;
      if (u + n == units) range[1] = w;
    }
    if (n > 0 || (shares == 0 && (!GROUPS || tokens > 0)))
      kv4_attend_token<T, HD, HEADS, GROUPS>(a, div, Kv4Job{t, (int64_t)w * group + t, tokens, L, u, u + n}, rest, lds);
    left -= n;
    if (left <= 0) break;
    u = 0;
    t += max(tokens, 1);
    __syncthreads();  // the next tokens' rows reuse the LDS
  }
}

// A workgroup of four waves joins four of a token's heads; tokens without keys get zeros.  A token that lies in one
// share is done.
template <typename T, int LANES, bool GROUPS>
__global__ __launch_bounds__(256) void kv4_join_kernel(const Kv4Args<T> a, int group, int blocks) {
  const int lane = threadIdx.x & 63;
  const int64_t t = blockIdx.x / blocks;
  const int h = (int)(blockIdx.x % blocks) * 4 + (threadIdx.x >> 6);
  if (h >= a.q_heads) return;
  int64_t t0 = t;  // where the token's group begins
  if constexpr (GROUPS) {
    const int32_t seq = a.qseq[t];
    while (t0 % group > 0 && a.qseq[t0 - 1] == seq) --t0;
  }
  T* out = a.out + (t * a.q_heads + h) * a.hd;
  if (kv4_group<GROUPS>(a, t0, group).units == 0) {
    for (int d = lane; d < a.hd; d += 64) out[d] = (T)0.0f;
    return;
  }
  const int w0 = a.range[2 * t], w1 = a.range[2 * t + 1];
  if (w0 == w1) return;
  const int64_t pi = ((int64_t)w0 * group + t) * a.q_heads + h, step = (int64_t)group * a.q_heads;
  join_states<T, LANES>(a.part + pi * a.hd, step * a.hd, a.states + 2 * pi, 2 * step, w1 - w0 + 1, out, a.hd);
}

// (token, head) rows of a sequence that go to the token kernel; fp32 tiles, with q and P in two parts each, take
// twice as long.
inline int kv4_few_rows(int dtype_bytes) { return dtype_bytes == 4 ? 64 : 32; }
// The kv heads that a workgroup takes side by side, and the workgroups that a token's (or share's) heads take.
inline int kv4_heads_side_by_side(int kv_heads, int hd) {
  return kv_heads % 8 == 0 && hd <= 128 ? 8 : kv_heads % 4 == 0 ? 4 : kv_heads % 2 == 0 ? 2 : 1;
}
inline int kv4_wgs_per_token(int q_heads, int kv_heads, int hd) {
  return kv_heads / kv4_heads_side_by_side(kv_heads, hd) * ((q_heads / kv_heads + 15) / 16);
}
// Shares of a call: the workgroups that the GPU's 1024 SIMDs hold at once (kv4_waves_per_simd), but no more than the
// block tables' keys make of kLeastShare units.  256 ragged sequences, 28 / 4 heads of 128, bf16: 512 shares 152 us,
// 768 145, 1024 147, 1536 159.  0: a workgroup for each token or group of tokens, where a batch is past kShareTokens
// or there is nothing to share.
inline int kv4_shares(int64_t tokens, int group, int q_heads, int kv_heads, int hd, int bs, int max_blocks,
                      int dtype_bytes) {
  if (tokens > (group > 1 ? kShareGroupTokens : kShareTokens)) return 0;
  const int64_t units = tokens * (((int64_t)bs * max_blocks + 31) / 32);
  const int side = kv4_heads_side_by_side(kv_heads, hd);
  const int waves = 1024 * kv4_waves_per_simd(hd * (dtype_bytes / 2), hd, side, group > 1);
  const int64_t wgs = waves / (side > 4 ? side : 4) / kv4_wgs_per_token(q_heads, kv_heads, hd);
  const int64_t n = std::min<int64_t>(std::max<int64_t>(1, wgs), units / kLeastShare);
  return units > INT32_MAX || n <= 1 ? 0 : (int)n;
}
inline int64_t kv4_slot_bytes(int q_heads, int hd) { return q_heads * (hd + 2) * (int64_t)sizeof(float); }
inline int64_t kv4_range_bytes(int64_t tokens) { return (2 * tokens + 3) / 4 * 16; }  // (in front of the slots)
inline int64_t kv4_part_bytes(int64_t tokens, int q_heads, int hd, int shares, int group) {
  return shares > 0 ? kv4_range_bytes(tokens) + ((int64_t)shares * group + tokens) * kv4_slot_bytes(q_heads, hd) : 0;
}

// The shares that a workspace has slots for: fewer where it is smaller than was asked for, but as many as there are
// groups of tokens to share out (a workgroup takes each of those by itself without), or none.
inline int kv4_fitting_shares(int shares, int64_t tokens, int q_heads, int hd, int group, int64_t ws_bytes) {
  const int64_t slots = (ws_bytes - kv4_range_bytes(tokens)) / kv4_slot_bytes(q_heads, hd);
  const int64_t n = std::min<int64_t>(shares, (slots - tokens) / group);
  return n > 1 && (n == shares || n * group >= tokens) ? (int)n : 0;
}

// The tokens of a launch: all, in shares or a workgroup each (tile_tokens = 0), or those from `first` on whose tiles
// are left.
struct Kv4Tokens {
  int shares, group;
  int64_t first, n;
  int tile_tokens;
};
template <typename T, int HD, int HEADS, bool GROUPS>
void launch_kv4_heads(const Kv4Args<T>& a, const Kv4Tokens& k, hipStream_t st) {
  using Lds = Kv4Lds<HD, HEADS>;
  static std::once_flag lds_once;
  std::call_once(lds_once, [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&kv4_token_kernel<T, HD, HEADS, GROUPS>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, Lds::kBytes);
  });
  const int64_t n = k.shares ? k.shares : (k.n + k.group - 1) / k.group * k.group;
  const dim3 grid((unsigned)(n * kv4_wgs_per_token(a.q_heads, a.kv_heads, HD)));
  kv4_token_kernel<T, HD, HEADS, GROUPS><<<grid, Lds::kWaves * 64, Lds::kBytes, st>>>(
      a, FastDiv((uint32_t)a.bs), k.shares, k.group, k.first, k.tile_tokens);
}
template <typename T, int HD, bool GROUPS>
int launch_kv4_groups(const Kv4Args<T>& a, const Kv4Tokens& k, hipStream_t st) {
  const int side = kv4_heads_side_by_side(a.kv_heads, HD);
  if constexpr (HD <= 128) {
    if (side == 8) launch_kv4_heads<T, HD, 8, GROUPS>(a, k, st);
  }
  if (side == 4) launch_kv4_heads<T, HD, 4, GROUPS>(a, k, st);
  else if (side == 2) launch_kv4_heads<T, HD, 2, GROUPS>(a, k, st);
  else if (side == 1) launch_kv4_heads<T, HD, 1, GROUPS>(a, k, st);
  const int rc = launch_status("paged_attention_kv4");
  if (rc != NVF_OK || k.shares == 0) return rc;
  const int blocks = (a.q_heads + 3) / 4;
  kv4_join_kernel<T, HD / 4, GROUPS><<<dim3((unsigned)(a.tokens * blocks)), 256, 0, st>>>(a, k.group, blocks);
  return launch_status("paged_attention_kv4(join)");
}
template <typename T, int HD>
int launch_kv4_token(const Kv4Args<T>& a, const Kv4Tokens& k, hipStream_t st) {
  return k.group > 1 ? launch_kv4_groups<T, HD, true>(a, k, st) : launch_kv4_groups<T, HD, false>(a, k, st);
}

// ---------------------------------------------------------------------------
// Several tokens of a sequence: the tiles of the 16-bit caches (attend_tile) in fp16, whose K and V rows a workgroup
// makes of the codes once for its 128 (token, head) rows.  A lane loads a quarter of a row (one scale) two or more
// steps ahead, and turns it into LDS rows in front of the barrier that hands them over.  K's eight dimensions of a
// dword lie in the codes' order 0 4 1 5 2 6 3 7, as q's operand does; V's in their own.
// P is rounded once to fp16 for 16-bit outputs, and kept in two parts for fp32: two parts would double the products
// of P . V, for an error of 2.1e-4 instead of 2.9e-4 in fp16.
// Chunks of 1000 and 700 tokens over 8192 and 4001 keys, 28 / 4 heads of 128, fp16: 250 us (token by token 1349) with
// the join of four key ranges, where the products alone take 106.  Matrix units busy a third of the cycles, vector
// instructions issued in half of them: rows are made of codes for each tile again, and the two do not overlap as they
// do over 16-bit rows.
template <typename T>
__device__ __forceinline__ void kv4_attend_row(const Kv4Args<T>& a, int c0, int c1, int seq, int64_t t, int h,
                                               int kvh, int L, int64_t split) {
  float m, l, acc[2];
  kv4_row_state<2>(a, c0, c1, 1, kChunk, seq, t, h, kvh, L, m, l, acc);
  const int lane = threadIdx.x & 63;
  const int64_t th = t * a.q_heads + h;
  for (int i = 0; i < 2; ++i) {
    const int d = lane + 64 * i;
    if (d >= a.hd) break;
    if (a.nsplit > 1) a.part[(th * a.nsplit + split) * a.hd + d] = acc[i];
    else a.out[th * a.hd + d] = from_f32<T>(l == 0.0f ? 0.0f : acc[i] / l);
  }
  if (a.nsplit > 1 && lane == 0) {
    float* ml = a.part + a.tokens * a.q_heads * a.nsplit * a.hd + 2 * (th * a.nsplit + split);
    ml[0] = m;
    ml[1] = l;
  }
}

template <typename T, int HD>
struct Kv4TileLoad {
  using Compute = _Float16;
  using Rows = TileRows<T, kCausalTile, _Float16>;
  using Lds = TileLds<_Float16, HD>;
  static constexpr int kQParts = sizeof(T) == 4 ? 2 : 1;
  static constexpr bool kTwoParts = sizeof(T) == 4, kEarly = true;
  static constexpr float kLazy = kKv4Lazy<T>, kLead = kKv4Lead<T>;
  static constexpr int kDwords = HD / 32;  // of codes: a lane's quarter of a row
  const Kv4Args<T>& a;
  Kv4Slabs table;
  uint8_t* lds;
  uint32_t code_off, word_off;
  uint32_t k_dst, v_dst;  // where the lane's first 16 bytes go, in buffer 0
  uint32_t kc[kDwords], kw, vc[kDwords], vw;
  int k_buf, v_buf;  // where the loaded ones belong; -1: there are none
  Kv4Magic magic;
  __device__ __forceinline__ Kv4TileLoad(const AttnArgs<T>& base, const FastDiv& div, const TileJob& job, const Rows& rows,
                                         int lane, int wave, uint8_t* lds_)
      : a(static_cast<const Kv4Args<T>&>(base)), table(a, div, rows.seq, rows.L_all), lds(lds_), k_buf(-1), v_buf(-1) {
    const int row = lane / 4, quarter = lane % 4;
    k_dst = (uint32_t)((16 * wave + row) * Lds::kRow + 16 * ((kDwords * quarter) ^ Lds::k_swz(row) ^ k_turn()));
    v_dst = (uint32_t)((16 * wave + row) * Lds::kRow + 16 * ((kDwords * quarter) ^ Lds::v_swz(row) ^ v_turn()));
    code_off = (uint32_t)row * table.row_b + (uint32_t)(job.kvh * (HD / 2)) + 4 * kDwords * quarter;
    word_off = (uint32_t)row * table.row_b + (uint32_t)(a.words + job.kvh * (HD / 16)) + 2 * (HD / 4 * quarter / kKv4Group);
  }
  // Dimension order of operand element j of eight: as kv4 codes unpack.  A row's largest value: in [2^10, 2^11).
  template <typename V8>
  static __device__ __forceinline__ float q(const AttnArgs<T>& a, const TileJob& job, const Rows& rows, int half,
                                            V8 (&qf)[kQParts][HD / 16]) {
    float x[HD / 16][8], most = 0.0f;
#pragma unroll
    for (int s = 0; s < HD / 16; ++s)
#pragma unroll
      for (int e = 0; e < 8; e += Pack<T>::N)
        Pack<T>::unpack(rows.ok ? ld16(a.q + (job.t0 + rows.ti) * a.q_stride + (int64_t)rows.head * HD + 16 * s +
                                       8 * half + e)
                                : u32x4{0, 0, 0, 0}, x[s] + e);
#pragma unroll
    for (int s = 0; s < HD / 16; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[s][e]));
    most = fmaxf(most, __shfl_xor(most, 32));
    const int shift = q_shift(most);
#pragma unroll
    for (int s = 0; s < HD / 16; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = ldexpf(x[s][(j >> 1) + 4 * (j & 1)], shift);
        qf[0][s][j] = (_Float16)v;
        if constexpr (kQParts == 2) qf[1][s][j] = rest_of(v, qf[0][s][j]);
      }
    return q_scale(a.scale_log2, shift);
  }
  __device__ __forceinline__ void load(const uint8_t* cache, const SlabEntry& e, uint32_t (&c)[kDwords], uint32_t& w) const {
    const __amdgpu_buffer_rsrc_t r = rows_rsrc(cache + table.at(e), table.bytes(e));
    if constexpr (kDwords == 2) {
      const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, code_off, 0, 0));
      c[0] = x[0];
      c[1] = x[1];
    } else {
      const u32x4 x = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, code_off, 0, 0));
#pragma unroll
      for (int i = 0; i < 4; ++i) c[i] = x[i];
    }
    w = __builtin_amdgcn_raw_buffer_load_b16(r, word_off, 0, 0);
  }
  __device__ __forceinline__ void k(const SlabEntry& e, int buf) {
    load(a.k, e, kc, kw);
    if (table.bad(e)) kw = kKv4NotANumber;  // keys without a block: NaN where they are seen
    k_buf = buf;
  }
  __device__ __forceinline__ void v(const SlabEntry& e, int buf) {
    load(a.v, e, vc, vw);
    v_buf = buf;
  }
  // Head size 128: the dword that a lane turns into its i-th store is i ^ turn, so that eight lanes (two rows) store
  // to distinct banks (k_swz has the row's lowest bit already): chunks in fp32 142 -> 136 us, fp16 the same within
  // 1%.  (64: 23.3 and 24.)
  static __device__ __forceinline__ int k_turn() { return kDwords == 4 ? (int)threadIdx.x & 2 : 0; }
  static __device__ __forceinline__ int v_turn() {
    return kDwords == 4 ? ((int)threadIdx.x & 2) | ((int)(threadIdx.x >> 2) & 1) : 0;
  }
  static __device__ __forceinline__ void turned(uint32_t (&c)[kDwords], int turn) {
    if constexpr (kDwords == 4) {
#pragma unroll
      for (int bit = 1; bit < kDwords; bit <<= 1) {
#pragma unroll
        for (int i = 0; i < kDwords; ++i) {
          if (i & bit) continue;
          const uint32_t x = c[i], y = c[i | bit];
          c[i] = turn & bit ? y : x;
          c[i | bit] = turn & bit ? x : y;
        }
      }
    }
  }
  // What is loaded, as LDS rows: 16-byte unit u of row r at position u ^ its swizzle (which the slab's first row does
  // not change, and of which V's has no low bits).
  __device__ __forceinline__ void commit() {
    if (k_buf >= 0) {
      const Kv4Half h = magic.half(kw | kw << 16);
      uint32_t dst = k_dst;
      asm volatile("" : "+v"(dst));  // (worked out here and not kept in registers through the chunks)
      turned(kc, k_turn());
#pragma unroll
      for (int i = 0; i < kDwords; ++i) st16(lds + (dst ^ (16u * i)) + k_buf * Lds::kBuf, magic.eight(kc[i], h));
    }
    if (v_buf >= 0) {
      const Kv4Half h = magic.half(vw | vw << 16);
      // a byte in both halves: its low nibble is the low half's value, the high one at bits 4 .. 7 the high half's
      const f16x2 z = {h.z_low[0], h.z_high[0]};
      uint32_t dst = v_dst;
      asm volatile("" : "+v"(dst));
      turned(vc, v_turn());
#pragma unroll
      for (int i = 0; i < kDwords; ++i) {
        u32x4 x;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const uint32_t both = __builtin_amdgcn_perm(0, vc[i], 0x0C000C00u + 0x00010001u * b);
          x[b] = __builtin_bit_cast(uint32_t, (__builtin_bit_cast(f16x2, (both & 0x00F0000Fu) | magic.mixed) + z) * h.d);
        }
        st16(lds + (dst ^ (16u * i)) + (2 + v_buf) * Lds::kBuf, x);
      }
    }
    k_buf = v_buf = -1;
  }
  // (The loads in flight are a lane's own: the barrier does not wait for them.)
  static __device__ __forceinline__ void hand_over() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  }
  static __device__ __forceinline__ void again(const AttnArgs<T>& base, const WindowRule&, const TileJob& job,
                                               const Rows& rows, uint64_t lanes, int wave) {
    const Kv4Args<T>& a = static_cast<const Kv4Args<T>&>(base);
    const int G = a.q_heads / a.kv_heads;
    for (uint64_t left = lanes & 0xFFFFFFFFu; left; left &= left - 1) {
      const int r = 32 * wave + __builtin_ctzll(left), i = r / G;
      kv4_attend_row(a, rows.c0, rows.c1, job.seq, job.t0 + i, job.kvh * G + (r - i * G), job.kvh, Rows::count(a, job, i),
                     job.state);
    }
  }
};

// Workgroup x = (tile, kv head), as window_tile_kernel's; tiles of many sequences are kv4_token_kernel's.
template <typename T, int HD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void kv4_tile_kernel(const Kv4Args<T> a,
                                                                                               const FastDiv div,
                                                                                               int tile_tokens, int tiles,
                                                                                               const SeqStarts seqs) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tile = tiles - 1 - (int)(blockIdx.x / a.kv_heads), kvh = (int)(blockIdx.x % a.kv_heads);
  TileAt at{0, 0, (int64_t)tile * tile_tokens};
  if (seqs.n > 0) at = tile_at(seqs.start, seqs.n, tile, tile_tokens);
  else at.n = a.tokens - at.t0 < tile_tokens ? (int)(a.tokens - at.t0) : tile_tokens;
  const TileRuns runs(a.qseq, at.t0, at.n);
  if (runs.count() > kTileMaxRuns) return;  // the whole workgroup: kv4_token_kernel's
  int r0 = 0;
#pragma unroll 1
  while (true) {
    const int r1 = runs.end_after(r0, at.n);
    const TileJob job{at.t0,     r0, r1, __builtin_amdgcn_readfirstlane(a.qseq[at.t0 + r0]), kvh, INT32_MAX,
                      (int)blockIdx.z, a.nsplit, blockIdx.z};
    attend_tile<T, HD, kCausalTile, Kv4TileLoad<T, HD>>(a, div, WindowRule{}, job, lds);
    r0 = r1;
    if (r0 >= at.n) break;
    __syncthreads();  // the next run's chunks reuse the LDS
  }
}

template <typename T>
void launch_kv4_any(const Kv4Args<T>& a, hipStream_t st) {
  const int G = a.q_heads / a.kv_heads;
  const auto by_group = [&](auto dpl) {
    constexpr int DPL = decltype(dpl)::value;
    const auto launch = [&](auto gh) {
      constexpr int GH = decltype(gh)::value;
      const dim3 grid((unsigned)(a.tokens * a.kv_heads * ((G + GH - 1) / GH)));
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

// How a call runs: tokens of a tile (0: none), and tokens that share a token kernel's columns.
struct Kv4Plan {
  int tile_tokens, group;
};
// Tiles, but for single tokens (promised, by the packing, or no more rows than one token's MFMAs take), head groups
// and sizes that tiles do not take, and sequences with few tokens each (`most`, by the packing on the host or the
// caller's promise; 0 unknown): a tile makes its rows of the codes whether its 128 rows are used or not, and leaves
// those of over kTileMaxRuns sequences; 16 columns read the codes again for each group of tokens.  32 sequences with
// 5 tokens of 4 heads each over up to 4096 keys: two groups 75 us, a tile 99; 128 of them 225 and 512.
inline Kv4Plan kv4_plan(int64_t tokens, int q_heads, int kv_heads, int hd, int64_t max_query_len, int64_t most,
                        int dtype_bytes) {
  const int G = q_heads / kv_heads;
  if (most == 1) max_query_len = 1;
  const int tq = hd == 64 || hd == 128 ? tiled_tokens(tokens, q_heads, kv_heads, max_query_len) : 0;
  // (no more than a sequence has, so that sequences of as many tokens begin where groups do)
  const int group = max_query_len == 1 || G > 8 ? 1 : (int)std::min<int64_t>(16 / G, most > 0 ? most : 16);
  if (tq == 0) return {0, group};
  return most > 0 && most * G <= kv4_few_rows(dtype_bytes) ? Kv4Plan{0, group} : Kv4Plan{tq, 1};
}
// The most tokens of a sequence, as far as the host knows.
inline int64_t kv4_most_tokens(const int32_t* cu, int num_seqs, int64_t max_query_len) {
  if (!cu) return max_query_len > 0 ? max_query_len : 0;
  int most = 0;
  for (int s = 0; s < num_seqs; ++s) most = std::max(most, cu[s + 1] - cu[s]);
  return most;
}
// Key ranges of tiles, where the host knows the packing.
inline int kv4_tile_split(int64_t tokens, int q_heads, int kv_heads, int hd, int bs, int max_blocks, int tile_tokens,
                          int64_t tiles) {
  const int64_t chunks = ((int64_t)bs * max_blocks + kChunk - 1) / kChunk;
  return tile_split(tiles * kv_heads, chunks, tokens * q_heads, hd, 2);
}

template <typename T, int HD>
int launch_kv4_tiles(Kv4Args<T> a, int tile_tokens, const int32_t* cu, void* ws, int64_t ws_bytes, hipStream_t st) {
  static std::once_flag lds_once;
  std::call_once(lds_once, [] {
    (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&kv4_tile_kernel<T, HD>),
                              hipFuncAttributeMaxDynamicSharedMemorySize, TileLds<_Float16, HD>::kBytes);
  });
  const TilePlan plan = cu ? tile_plan(cu, a.num_seqs, tile_tokens) : TilePlan{};
  const int tiles = plan.seqs.n > 0 ? tiles_of(plan.seqs.start, plan.seqs.n, tile_tokens)
                                    : (int)((a.tokens + tile_tokens - 1) / tile_tokens);
  if (plan.seqs.n > 0) {  // (without the packing single tokens may be left, which write whole results)
    const int nsplit = kv4_tile_split(a.tokens, a.q_heads, a.kv_heads, HD, a.bs, a.max_blocks, tile_tokens, tiles);
    a.part = static_cast<float*>(ws);
    const int64_t one = a.tokens * a.q_heads * (HD + 2) * (int64_t)sizeof(float);  // a range's states
    a.nsplit = ws ? (int)std::max<int64_t>(1, std::min<int64_t>(nsplit, ws_bytes / one)) : 1;
  }
  const dim3 grid((unsigned)(tiles * a.kv_heads), 1, (unsigned)a.nsplit);
  kv4_tile_kernel<T, HD><<<grid, 256, TileLds<_Float16, HD>::kBytes, st>>>(a, FastDiv((uint32_t)a.bs), tile_tokens,
                                                                           tiles, plan.seqs);
  const int rc = launch_status("paged_attention_kv4");
  if (rc != NVF_OK) return rc;
  if (a.nsplit > 1) return launch_attn_join(a, "paged_attention_kv4(join)", st);
  const Kv4Tokens left{0, 1, plan.known ? plan.first : 0, plan.known ? plan.end - plan.first : a.tokens, tile_tokens};
  return left.n > 0 ? launch_kv4_token<T, HD>(a, left, st) : NVF_OK;
}

template <typename T>
int kv4_dispatch(Kv4Args<T> a, int64_t max_query_len, const int32_t* cu, void* ws, int64_t ws_bytes, hipStream_t st) {
  const bool mfma = kv4_mfma_shape(a.hd, a.bs) && aligned16(a.q) && aligned16(a.out) && a.q_stride % Pack<T>::N == 0 &&
                    a.scale_log2 > 0.0f && a.row_bytes < INT32_MAX / 64 && a.num_blocks <= INT32_MAX / a.bs;
  if (!mfma) {
    launch_kv4_any(a, st);
    return launch_status("paged_attention_kv4");
  }
  const Kv4Plan plan = kv4_plan(a.tokens, a.q_heads, a.kv_heads, a.hd, max_query_len,
                                kv4_most_tokens(cu, a.num_seqs, max_query_len), (int)sizeof(T));
  if (plan.tile_tokens)
    return a.hd == 64 ? launch_kv4_tiles<T, 64>(a, plan.tile_tokens, cu, ws, ws_bytes, st)
                      : launch_kv4_tiles<T, 128>(a, plan.tile_tokens, cu, ws, ws_bytes, st);
  Kv4Tokens all{0, plan.group, 0, a.tokens, 0};
  all.shares = kv4_shares(a.tokens, all.group, a.q_heads, a.kv_heads, a.hd, a.bs, a.max_blocks, (int)sizeof(T));
  all.shares = kv4_fitting_shares(all.shares, a.tokens, a.q_heads, a.hd, all.group, ws ? ws_bytes : 0);
  if (all.shares > 0) {
    a.range = static_cast<int32_t*>(ws);
    a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kv4_range_bytes(a.tokens));
    a.states = a.part + ((int64_t)all.shares * all.group + a.tokens) * a.q_heads * a.hd;
  }
  return a.hd == 64    ? launch_kv4_token<T, 64>(a, all, st)
         : a.hd == 128 ? launch_kv4_token<T, 128>(a, all, st)
                       : launch_kv4_token<T, 256>(a, all, st);
}

}  // namespace nvf

using namespace nvf;

extern "C" {

int64_t nvf_paged_attention_kv4_workspace_size(int64_t tokens, int q_heads, int kv_heads, int head_dim, int block_size,
                                               int max_blocks, int64_t max_query_len) {
  if (tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || !kv4_head_dim_ok(head_dim) || block_size <= 0 || max_blocks <= 0 ||
      q_heads % kv_heads)
    return 0;
  if (!kv4_mfma_shape(head_dim, block_size)) return 0;
  // (The packing is not known here: the largest of what tiles, groups of tokens and single ones need, whatever
  // max_query_len says but that no sequence has more.  Fewer tiles mean more key ranges, and no packing has fewer;
  // 16-bit types have as many shares as fp32, or more.)
  const int64_t most = std::max(1, kv4_few_rows(4) / (q_heads / kv_heads));  // that go to the token kernel
  const Kv4Plan few = kv4_plan(tokens, q_heads, kv_heads, head_dim, max_query_len,
                               max_query_len > 0 ? std::min(max_query_len, most) : most, 4);
  const Kv4Plan many = kv4_plan(tokens, q_heads, kv_heads, head_dim, max_query_len, std::max<int64_t>(max_query_len, 0), 2);
  const auto of_tokens = [&](int group) {
    const int shares = kv4_shares(tokens, group, q_heads, kv_heads, head_dim, block_size, max_blocks, 2);
    return kv4_part_bytes(tokens, q_heads, head_dim, shares, group);
  };
  int64_t bytes = std::max(of_tokens(1), few.tile_tokens ? 0 : of_tokens(few.group));
  if (many.tile_tokens) {
    const int64_t tiles = (tokens + many.tile_tokens - 1) / many.tile_tokens;
    const int nsplit = kv4_tile_split(tokens, q_heads, kv_heads, head_dim, block_size, max_blocks, many.tile_tokens, tiles);
    bytes = std::max(bytes, part_bytes(tokens, q_heads, head_dim, nsplit));
  }
  return bytes;
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
    rc = kv4_dispatch<T>(a, max_query_len, cu_seqlens_host, workspace, workspace_bytes, as_stream(stream));
  });
  return rc;
}

}  // extern "C"
