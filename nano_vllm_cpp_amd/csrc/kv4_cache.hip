// Keys and values appended to a 4-bit paged cache (kv4.hpp), with the per-head norm and the rotation
// applied on the way, and its rows read back as values.
//
//   q          as nvf_rotary: fp32 math, one rounding
//   k          the same in 64 bits, then each 32 dimensions to a scale, a zero point and codes
//   v          its values as they are, likewise
//
// Codes are whole numbers: a key that fp32 arithmetic put on the other side of a border between two
// codes would be off by a whole step.  In 64 bits that happens to one value in about 2^45.  fp64 runs at
// half the rate of fp32, and memory still bounds the call: 16384 tokens of 28 / 4 heads of 128 in bf16
// take 57 us, 52 into 16-bit caches, for bytes that a copy moves in 42.
// Calls of a few hundred tokens take as long as their launch, 9 us.
#include <math.h>

#include <algorithm>

#include "kv4.hpp"
#include "rotary.hpp"

namespace nvf {

constexpr int kKv4Threads = 256;

template <typename T>
struct Kv4StoreArgs {
  const T* q;
  T* q_out;
  const T* k;
  T* k_out;
  const T* v;
  uint8_t* kc;
  uint8_t* vc;
  const int64_t* positions;
  const double* inv_freq;
  const T* qw;
  const T* kw;
  const int32_t* slots;
  int64_t tokens, cache_rows, row_bytes;
  int64_t q_stride, q_out_stride, k_stride, k_out_stride, v_stride;
  int q_heads, kv_heads, hd, rot;
  double attn_scale, eps;
  bool interleaved;
};

// A wave's sum, in 64 bits.
__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

// Head sizes of 32 to 256 (multiples of 32), any stride and alignment: a wave per (token, head), heads q, then
// k, then v.  A head lies in LDS in 64 bits; half a wave takes 32 dimensions at a time to their codes.
template <typename T>
__global__ __launch_bounds__(kKv4Threads) void kv4_store_any_kernel(const Kv4StoreArgs<T> a) {
  __shared__ double head[kKv4Threads / 64][2 * kRotMaxPairs];
  const int heads = a.q_heads + 2 * a.kv_heads, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t item = (int64_t)blockIdx.x * (kKv4Threads / 64) + w;
  const bool some = item < a.tokens * heads;  // (every wave meets the barriers)
  const int64_t t = some ? item / heads : 0;
  const int h = some ? (int)(item - t * heads) : 0;
  const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
  const int hk = is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads;
  const T* x = is_q   ? a.q + t * a.q_stride + (int64_t)h * a.hd
               : is_v ? a.v + t * a.v_stride + (int64_t)hk * a.hd
                      : a.k + t * a.k_stride + (int64_t)hk * a.hd;
  double* y = head[w];
  if (some)
    for (int d = lane; d < a.hd; d += 64) y[d] = (double)to_f32(x[d]);
  __syncthreads();
  if (some && !is_v) {
    const T* gamma = is_q ? a.qw : a.kw;
    T* out = is_q ? a.q_out + t * a.q_out_stride + (int64_t)h * a.hd
                  : a.k_out ? a.k_out + t * a.k_out_stride + (int64_t)hk * a.hd : nullptr;
    if (gamma) {
      double ss = 0.0;
      for (int d = lane; d < a.hd; d += 64) ss = fma(y[d], y[d], ss);
      const double inv = 1.0 / sqrt(wave_sum64(ss) / (double)a.hd + a.eps);
      for (int d = lane; d < a.hd; d += 64) y[d] = y[d] * inv * (double)to_f32(gamma[d]);
      __builtin_amdgcn_wave_barrier();
    }
    const int64_t position = a.positions[t];
    for (int i = lane; i < a.rot / 2; i += 64) {
      const int da = a.interleaved ? 2 * i : i, db = a.interleaved ? 2 * i + 1 : i + a.rot / 2;
      const Turn64 turn = rotary_cs64(position, a.inv_freq[i], a.attn_scale);
      const double x1 = y[da], x2 = y[db];
      y[da] = x1 * turn.c - x2 * turn.s;
      y[db] = x2 * turn.c + x1 * turn.s;
    }
    __builtin_amdgcn_wave_barrier();
    if (out)
      for (int d = lane; d < a.hd; d += 64) out[d] = (T)y[d];
  }
  __syncthreads();
  if (!some || is_q) return;
  const int32_t slot = a.slots[t];
  if (slot < 0 || slot >= a.cache_rows) return;
  uint8_t* row = (is_v ? a.vc : a.kc) + slot * a.row_bytes;
  const int words = a.hd / kKv4Group, half = lane >> 5, l32 = lane & 31;
  for (int g = half; g < words; g += 2) {
    const double v = y[kKv4Group * g + l32];
    double low = fmin(v, 0.0), high = fmax(v, 0.0);
    int odd = !isfinite(v);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      low = fmin(low, __shfl_xor(low, d));
      high = fmax(high, __shfl_xor(high, d));
      odd |= __shfl_xor(odd, d);
    }
    Kv4Scale s = kv4_scale_of(low, high);
    if (odd) s = Kv4Scale{0.0, 0.0, kKv4NotANumber};
    const uint32_t code = odd ? 0 : kv4_code<double>(v, s.d, s.z, s.inverse()), next = __shfl_down(code, 1);
    if (l32 % 2 == 0) row[(int64_t)hk * (a.hd / 2) + 16 * g + l32 / 2] = (uint8_t)(code | next << 4);
    if (l32 == 0)
      *reinterpret_cast<uint16_t*>(row + (int64_t)a.kv_heads * (a.hd / 2) + 2 * (hk * words + g)) = (uint16_t)s.word;
  }
}

// 16-byte rows of head sizes 64, 128 and 256: a workgroup takes `per` tokens, whose (cos, sin) pairs go into LDS once
// for all heads, in 64 bits for the keys and in 32 for q.  A head of q is HD / 2 / N lanes of two 16-byte vectors
// each, so that a pair's two values are one lane's.  A head of k or v is HD / 8 lanes of eight consecutive
// dimensions, a dword of codes each, four lanes a scale; a lane of k reads the eight dimensions that its own pair
// with as well.  (With both caches read back 16384 tokens take 67 us, a head a wave 294; v's codes in 64 bits, in k's
// loop, 75.)
constexpr int kKv4MaxTokens = 4;

template <typename T, typename F>
__device__ __forceinline__ void unpack8(const u32x4* x, F (&y)[8]) {
  constexpr int N = Pack<T>::N;
  float f[8];
#pragma unroll
  for (int e = 0; e < 8 / N; ++e) Pack<T>::unpack(x[e], f + N * e);
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = (F)f[j];
}
// Another lane's value of the four that share a scale.
template <int CTRL, typename F>
__device__ __forceinline__ F quad_mov(F v) {
  if constexpr (sizeof(F) == 8) {
    const u32x2 w = __builtin_bit_cast(u32x2, v);
    const uint32_t lo = w[0], hi = w[1];  // (a bit_cast of a vector's element reads element 0)
    const float l = dpp_mov<CTRL>(__builtin_bit_cast(float, lo)), h = dpp_mov<CTRL>(__builtin_bit_cast(float, hi));
    return __builtin_bit_cast(F, u32x2{__builtin_bit_cast(uint32_t, l), __builtin_bit_cast(uint32_t, h)});
  } else {
    return dpp_mov<CTRL>(v);
  }
}
// The codes of this lane's eight of a group's 32 values, and the group's word.  (The least and the largest value are
// exact in F; their scale is worked out in 64 bits.)
template <typename F>
__device__ __forceinline__ uint32_t kv4_eight_codes(const F (&y)[8], uint32_t& word) {
  F low = 0, high = 0, odd = 0;  // odd: NaN if one of the values is no finite number
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    low = __builtin_elementwise_min(low, y[j]);
    high = __builtin_elementwise_max(high, y[j]);
    odd = __builtin_elementwise_fma(y[j], (F)0, odd);
  }
  low = __builtin_elementwise_min(low, quad_mov<0xb1>(low));
  high = __builtin_elementwise_max(high, quad_mov<0xb1>(high));
  odd += quad_mov<0xb1>(odd);
  low = __builtin_elementwise_min(low, quad_mov<0x4e>(low));
  high = __builtin_elementwise_max(high, quad_mov<0x4e>(high));
  odd += quad_mov<0x4e>(odd);
  const Kv4Scale s = kv4_scale_of((double)low, (double)high);
  const F d = (F)s.d, z = (F)s.z, inv = (F)s.inverse();
  uint32_t codes = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) codes |= kv4_code<F>(y[j], d, z, inv) << (4 * j);
  const bool fine = odd == (F)0;
  word = fine ? s.word : kKv4NotANumber;
  return fine ? codes : 0;
}

template <typename T, int HD, bool INTERLEAVED>
__global__ __launch_bounds__(kKv4Threads) void kv4_store_vec_kernel(const Kv4StoreArgs<T> a, const FastDiv q_div,
                                                                    const FastDiv kv_div, int per) {
  constexpr int N = Pack<T>::N, LPH = HD / 2 / N, kHeads = kKv4Threads / LPH, kLanes = HD / 8;
  __shared__ Turn64 cs64[kKv4MaxTokens * HD / 2];
  __shared__ float2 cs32[kKv4MaxTokens * HD / 2];
  const int half = a.rot / 2;
  const int64_t t0 = (int64_t)blockIdx.x * per;
  const int n = a.tokens - t0 < per ? (int)(a.tokens - t0) : per;

  // q: this lane's vectors of a head, and whether they turn
  const int sub = threadIdx.x % LPH, items = n * a.q_heads;
  int d1 = 2 * sub * N, d2 = d1 + N;
  bool turn1 = d1 < a.rot, turn2 = d2 < a.rot;
  if constexpr (!INTERLEAVED) {
    turn1 = turn2 = sub * N < half;
    if (turn1) {
      d1 = sub * N;
      d2 = d1 + half;
    }  // else: past the rotated dimensions, where 2 sub N >= rot
  }
  struct Item {
    int i, h;
    u32x4 x1, x2;
  };
  const auto load_q = [&](int at) {
    Item it{};
    it.i = (int)q_div.div((uint32_t)at);
    it.h = at - it.i * a.q_heads;
    const T* x = a.q + (t0 + it.i) * a.q_stride + (int64_t)it.h * HD;
    it.x1 = ld16_nt(x + d1);
    it.x2 = ld16_nt(x + d2);
    return it;
  };
  // k and v: eight dimensions from d0 on, and those of k that they pair with
  const int kv_sub = threadIdx.x % kLanes, d0 = 8 * kv_sub;
  const bool turns = d0 < a.rot;
  const int pair0 = INTERLEAVED || !turns ? d0 : d0 < half ? d0 + half : d0 - half;
  constexpr int kVecs = 8 / N, kKvHeads = kKv4Threads / kLanes;
  struct KvItem {
    int i, h, slot;
    u32x4 x[kVecs];
  };
  const int kv_items = n * a.kv_heads;
  const auto load_kv = [&](const T* rows, int64_t stride, int at) {
    KvItem it{};
    it.i = (int)kv_div.div((uint32_t)at);
    it.h = at - it.i * a.kv_heads;
    const T* x = rows + (t0 + it.i) * stride + (int64_t)it.h * HD + d0;
#pragma unroll
    for (int e = 0; e < kVecs; ++e) it.x[e] = ld16(x + N * e);
    it.slot = a.slots[t0 + it.i];
    return it;
  };
  // eight codes and, of every fourth lane, the word
  const auto store = [&](uint8_t* cache, const KvItem& it, uint32_t codes, uint32_t word) {
    if (it.slot < 0 || it.slot >= a.cache_rows) return;
    uint8_t* row = cache + it.slot * a.row_bytes;
    *reinterpret_cast<uint32_t*>(row + it.h * (HD / 2) + 4 * kv_sub) = codes;
    if (kv_sub % 4 == 0)
      *reinterpret_cast<uint16_t*>(row + a.kv_heads * (HD / 2) + 2 * (it.h * (HD / 32) + kv_sub / 4)) = (uint16_t)word;
  };

  int at = threadIdx.x / LPH, kv_at = threadIdx.x / kLanes;
  Item it{};
  KvItem key{}, value{};
  if (at < items) it = load_q(at);
  if (kv_at < kv_items) {
    key = load_kv(a.k, a.k_stride, kv_at);
    value = load_kv(a.v, a.v_stride, kv_at);
  }
  for (int i = threadIdx.x; i < n * half; i += kKv4Threads) {
    const int tk = i / half;
    const Turn64 turn = rotary_cs64(a.positions[t0 + tk], a.inv_freq[i - tk * half], a.attn_scale);
    cs64[i] = turn;
    cs32[i] = float2{(float)turn.c, (float)turn.s};
  }
  __syncthreads();

  for (; at < items; at += kHeads) {
    Item next{};
    if (at + kHeads < items) next = load_q(at + kHeads);
    float x1[N], x2[N];
    Pack<T>::unpack(it.x1, x1);
    Pack<T>::unpack(it.x2, x2);
    if (a.qw) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) ss = fmaf(x1[j], x1[j], fmaf(x2[j], x2[j], ss));
      const float inv = 1.0f / sqrtf(group_sum<LPH>(ss) / (float)HD + (float)a.eps);
      float w1[N], w2[N];
      Pack<T>::unpack(ld16(a.qw + d1), w1);
      Pack<T>::unpack(ld16(a.qw + d2), w2);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x1[j] = x1[j] * inv * w1[j];
        x2[j] = x2[j] * inv * w2[j];
      }
    }
    const float2* c = cs32 + it.i * half;
    if constexpr (INTERLEAVED) {
      const auto turn = [&](float* x, int d) {
#pragma unroll
        for (int j = 0; j < N; j += 2) {
          const float2 r = c[(d + j) / 2];
          const float p = x[j], q = x[j + 1];
          x[j] = p * r.x - q * r.y;
          x[j + 1] = q * r.x + p * r.y;
        }
      };
      if (turn1) turn(x1, d1);
      if (turn2) turn(x2, d2);
    } else if (turn1) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float2 r = c[d1 + j];
        const float p = x1[j], q = x2[j];
        x1[j] = p * r.x - q * r.y;
        x2[j] = q * r.x + p * r.y;
      }
    }
    T* y = a.q_out + (t0 + it.i) * a.q_out_stride + (int64_t)it.h * HD;
    st16_nt(y + d1, Pack<T>::pack(x1));
    st16_nt(y + d2, Pack<T>::pack(x2));
    it = next;
  }

  for (int x = kv_at; x < kv_items; x += kKvHeads) {
    KvItem next{};
    if (x + kKvHeads < kv_items) next = load_kv(a.k, a.k_stride, x + kKvHeads);
    double y[8];
    unpack8<T>(key.x, y);
    double inv = 1.0;
    if (a.kw) {
      double ss = 0.0;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss = fma(y[j], y[j], ss);
#pragma unroll
      for (int d = 1; d < kLanes; d <<= 1) ss += __shfl_xor(ss, d);
      inv = 1.0 / sqrt(ss / (double)HD + a.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = y[j] * inv * (double)to_f32(a.kw[d0 + j]);
    }
    if (turns) {
      const Turn64* c = cs64 + key.i * half;
      if constexpr (INTERLEAVED) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const Turn64 r = c[(d0 + j) / 2];
          const double x1 = y[j], x2 = y[j + 1];
          y[j] = x1 * r.c - x2 * r.s;
          y[j + 1] = x2 * r.c + x1 * r.s;
        }
      } else {
        const bool low = d0 < half;
        const T* other = a.k + (t0 + key.i) * a.k_stride + (int64_t)key.h * HD + pair0;  // (read by this wave a moment ago)
        u32x4 px[kVecs];
#pragma unroll
        for (int e = 0; e < kVecs; ++e) px[e] = ld16(other + N * e);
        double z[8];
        unpack8<T>(px, z);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (a.kw) z[j] = z[j] * inv * (double)to_f32(a.kw[pair0 + j]);
          const Turn64 r = c[(low ? d0 : pair0) + j];
          y[j] = y[j] * r.c + z[j] * (low ? -r.s : r.s);
        }
      }
    }
    if (a.k_out) {  // rounded to fp32 and then to T: half a step of T and 2^-24 of it
      T* out = a.k_out + (t0 + key.i) * a.k_out_stride + (int64_t)key.h * HD + d0;
#pragma unroll
      for (int e = 0; e < kVecs; ++e) {
        float f[N];
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = (float)y[N * e + j];
        st16(out + N * e, Pack<T>::pack(f));
      }
    }
    uint32_t word;
    const uint32_t codes = kv4_eight_codes(y, word);
    store(a.kc, key, codes, word);
    key = next;
  }
  using F = std::conditional_t<sizeof(T) == 4, double, float>;
  for (int x = kv_at; x < kv_items; x += kKvHeads) {
    KvItem next{};
    if (x + kKvHeads < kv_items) next = load_kv(a.v, a.v_stride, x + kKvHeads);
    F y[8];
    unpack8<T>(value.x, y);
    uint32_t word;
    const uint32_t codes = kv4_eight_codes(y, word);
    store(a.vc, value, codes, word);
    value = next;
  }
}

template <typename T, int HD>
void launch_kv4_store_vec(const Kv4StoreArgs<T>& a, hipStream_t st) {
  constexpr int LPH = HD / 2 / Pack<T>::N;
  // tokens of a workgroup: enough heads for its threads, and a few passes of them where there are many tokens
  const int fill = (kKv4Threads + a.q_heads * LPH - 1) / (a.q_heads * LPH);
  const int per = (int)std::min<int64_t>(kKv4MaxTokens, std::max<int64_t>(fill, a.tokens / 2048));
  const dim3 grid((unsigned)((a.tokens + per - 1) / per));
  const FastDiv q_div((uint32_t)a.q_heads), kv_div((uint32_t)a.kv_heads);
  if (a.interleaved) kv4_store_vec_kernel<T, HD, true><<<grid, kKv4Threads, 0, st>>>(a, q_div, kv_div, per);
  else kv4_store_vec_kernel<T, HD, false><<<grid, kKv4Threads, 0, st>>>(a, q_div, kv_div, per);
}

template <typename T>
int kv4_store_dispatch(const Kv4StoreArgs<T>& a, hipStream_t st) {
  constexpr int N = Pack<T>::N;
  const auto rows16 = [](const void* p, int64_t stride) { return !p || (aligned16(p) && stride % N == 0); };
  const bool vec = (a.interleaved ? a.rot : a.rot / 2) % 8 == 0 && rows16(a.q, a.q_stride) &&
                   rows16(a.q_out, a.q_out_stride) && rows16(a.k, a.k_stride) && rows16(a.k_out, a.k_out_stride) &&
                   rows16(a.v, a.v_stride) && rows16(a.qw, 0) && rows16(a.kw, 0);
  if (vec && a.hd == 64) launch_kv4_store_vec<T, 64>(a, st);
  else if (vec && a.hd == 128) launch_kv4_store_vec<T, 128>(a, st);
  else if (vec && a.hd == 256) launch_kv4_store_vec<T, 256>(a, st);
  else {
    const int64_t items = a.tokens * (a.q_heads + 2 * a.kv_heads), waves = kKv4Threads / 64;
    kv4_store_any_kernel<T><<<dim3((unsigned)((items + waves - 1) / waves)), kKv4Threads, 0, st>>>(a);
  }
  return launch_status("rotary_store_kv4");
}

// Values of eight dimensions at a time: a dword of codes, one or two 16-byte stores.  A workgroup takes `per` rows.
// Bound by its bytes: 16384 rows of 4 heads of 128 to bf16 6.2 us with its launch (a copy's rate alone 3.2).
template <typename T>
__global__ __launch_bounds__(kKv4Threads) void kv4_unpack_kernel(const uint8_t* __restrict__ cache, T* __restrict__ out,
                                                                 int64_t rows, int64_t row_bytes, int per,
                                                                 const FastDiv row_dwords) {
  constexpr int N = Pack<T>::N;
  const int dwords = (int)row_dwords.d;  // of a row's codes
  const int64_t r0 = (int64_t)blockIdx.x * per;
  const int n = (int)(rows - r0 < per ? rows - r0 : per) * dwords;
  for (int i = threadIdx.x; i < n; i += kKv4Threads) {
    const int r = (int)row_dwords.div((uint32_t)i), at = i - r * dwords;
    const uint8_t* p = cache + (r0 + r) * row_bytes;
    const uint32_t codes = *reinterpret_cast<const uint32_t*>(p + 4 * at);
    const uint32_t word = *reinterpret_cast<const uint16_t*>(p + 4 * dwords + 2 * (at / 4));
    const float d = kv4_scale(word);
    const int z = (int)(word & 15u);
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = d * (float)((int)(codes >> (4 * e) & 15u) - z);
    T* o = out + ((r0 + r) * dwords + at) * 8;
#pragma unroll
    for (int e = 0; e < 8; e += N) st16_nt(o + e, Pack<T>::pack(f + e));
  }
}

}  // namespace nvf

using namespace nvf;

extern "C" {

int64_t nvf_kv4_row_bytes(int kv_heads, int head_dim) {
  return kv_heads > 0 && kv4_head_dim_ok(head_dim) ? kv4_row_bytes(kv_heads, head_dim) : 0;
}

int nvf_rotary_store_kv4(const void* q, void* q_out, const void* k, void* k_out, const void* v,
                         const int64_t* positions, const double* inv_freq, int interleaved, int rotary_dim,
                         double attn_scale, const void* q_w, const void* k_w, double eps, int64_t tokens, int q_heads,
                         int kv_heads, int head_dim, int64_t q_stride, int64_t q_out_stride, int64_t k_stride,
                         int64_t k_out_stride, int64_t v_stride, void* k_cache, void* v_cache,
                         const int32_t* slot_mapping, int64_t cache_rows, int dtype, void* stream) {
  const char* who = "nvf_rotary_store_kv4";
  if (!kv4_head_dim_ok(head_dim))
    return fail(NVF_ERR_INVALID, "%s: head_dim=%d is not a multiple of %d up to 256", who, head_dim, kKv4Group);
  if (tokens != 0 && !k_cache) return fail(NVF_ERR_INVALID, "%s: NULL pointer", who);
  const int rc0 = check_rotary(who, q, q_out, k, k_out, v, positions, inv_freq, rotary_dim, q_w, k_w, tokens, q_heads,
                               kv_heads, head_dim, q_stride, q_out_stride, k_stride, k_out_stride, v_stride,
                               tokens != 0, v_cache, slot_mapping, cache_rows, dtype);
  if (rc0 != NVF_OK || tokens == 0) return rc0;
  if (!aligned16(k_cache) || !aligned16(v_cache))
    return fail(NVF_ERR_INVALID, "%s: the caches must be 16-byte aligned", who);
  cache_rows = cache_rows < ((int64_t)1 << 31) ? cache_rows : (int64_t)1 << 31;  // (as many as slots name)
  const int64_t row_bytes = kv4_row_bytes(kv_heads, head_dim), cache_bytes = cache_rows * row_bytes;
  if (bytes_overlap(k_cache, cache_bytes, v_cache, cache_bytes))
    return fail(NVF_ERR_INVALID, "%s: k_cache overlaps v_cache", who);
  if (tokens * (q_heads + 2 * (int64_t)kv_heads) > INT32_MAX) return fail(NVF_ERR_INVALID, "%s: too many heads", who);
  int rc = NVF_OK;
  NVF_DISPATCH_DTYPE(dtype, T, {
    Kv4StoreArgs<T> a{};
    a.q = static_cast<const T*>(q);
    a.q_out = static_cast<T*>(q_out);
    a.k = static_cast<const T*>(k);
    a.k_out = static_cast<T*>(k_out);
    a.v = static_cast<const T*>(v);
    a.kc = static_cast<uint8_t*>(k_cache);
    a.vc = static_cast<uint8_t*>(v_cache);
    a.positions = positions;
    a.inv_freq = inv_freq;
    a.qw = static_cast<const T*>(q_w);
    a.kw = static_cast<const T*>(k_w);
    a.slots = slot_mapping;
    a.tokens = tokens;
    a.cache_rows = cache_rows;
    a.row_bytes = row_bytes;
    a.q_stride = q_stride;
    a.q_out_stride = q_out_stride;
    a.k_stride = k_stride;
    a.k_out_stride = k_out_stride;
    a.v_stride = v_stride;
    a.q_heads = q_heads;
    a.kv_heads = kv_heads;
    a.hd = head_dim;
    a.rot = rotary_dim;
    a.attn_scale = attn_scale;
    a.eps = eps;
    a.interleaved = interleaved != 0;
    rc = kv4_store_dispatch<T>(a, as_stream(stream));
  });
  return rc;
}

int nvf_kv4_unpack(const void* cache, void* out, int64_t rows, int kv_heads, int head_dim, int dtype, void* stream) {
  const char* who = "nvf_kv4_unpack";
  if (!dtype_ok(dtype)) return fail(NVF_ERR_INVALID, "%s: bad dtype %d", who, dtype);
  if (rows < 0 || kv_heads <= 0 || !kv4_head_dim_ok(head_dim) || (int64_t)kv_heads * head_dim > 1 << 20)
    return fail(NVF_ERR_INVALID, "%s: bad shape rows=%lld kv_heads=%d head_dim=%d", who, (long long)rows, kv_heads,
                head_dim);
  if (rows == 0) return NVF_OK;
  if (!cache || !out) return fail(NVF_ERR_INVALID, "%s: NULL pointer", who);
  if (!aligned16(cache) || !aligned16(out)) return fail(NVF_ERR_INVALID, "%s: not 16-byte aligned", who);
  const int64_t row_bytes = kv4_row_bytes(kv_heads, head_dim), values = (int64_t)kv_heads * head_dim;
  const int dwords = (int)(values / 8);
  const int per = (2048 + dwords - 1) / dwords;
  const int64_t blocks = (rows - 1) / per + 1;
  if (blocks > INT32_MAX / kKv4Threads) return fail(NVF_ERR_INVALID, "%s: too many rows", who);
  if (bytes_overlap(cache, rows * row_bytes, out, rows * values * dtype_bytes(dtype)))
    return fail(NVF_ERR_INVALID, "%s: out overlaps the cache", who);
  NVF_DISPATCH_DTYPE(dtype, T, (kv4_unpack_kernel<T><<<dim3((unsigned)blocks), kKv4Threads, 0, as_stream(stream)>>>(
                                   static_cast<const uint8_t*>(cache), static_cast<T*>(out), rows, row_bytes, per,
                                   FastDiv((uint32_t)dwords))));
  return launch_status("kv4_unpack");
}

}  // extern "C"
