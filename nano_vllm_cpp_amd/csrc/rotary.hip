// Rotary positions for long contexts: half or interleaved pairs, the first rotary_dim dimensions
// of each head, frequencies and angles in fp64, with the optional per-head norm before and the KV
// store after.
//
//   pair i of a head: (a, b) = dims (i, i + rotary_dim / 2), or (2 i, 2 i + 1) interleaved
//   (a, b) <- s (a cos - b sin, b cos + a sin),  angle = position * inv_freq[i], s = attn_scale
//
// The angle is a product in fp64 reduced to [-pi, pi] there: position 10^6 in fp32 would leave an
// angle of 10^6 with an error of 0.03.
#include <math.h>

#include <algorithm>

#include "nvf_device.hpp"
#include "nvf_host.hpp"

namespace nvf {

constexpr int kRotThreads = 256;
constexpr int kRotMaxPairs = 128;  // of a head: head_dim <= 256

template <typename T>
struct RotaryArgs {
  const T* q;
  T* q_out;
  const T* k;
  T* k_out;
  const T* v;
  T* kc;
  T* vc;
  const int64_t* positions;
  const double* inv_freq;
  const T* qw;
  const T* kw;
  const int32_t* slots;
  int64_t tokens, cache_rows;
  int64_t q_stride, q_out_stride, k_stride, k_out_stride, v_stride;
  int q_heads, kv_heads, hd, rot;
  float attn_scale, eps;
  bool interleaved;
};

// (cos, sin) of position * freq, times the scale.  The fp32 functions take the reduced angle rounded to fp32, which is off
// by up to 2^-23; what the rounding left, d, turns the result back: cos(f + d) = cos f - d sin f, and d^2 is below 2^-46.
__device__ __forceinline__ float2 rotary_cs(int64_t position, double freq, float scale) {
  const double t = (double)position * freq;
  const double n = rint(t * 0.15915494309189535);                             // 1 / (2 pi)
  const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, t));  // 2 pi in two parts
  const float f = (float)r, d = (float)(r - (double)f);
  float sn, cs;
  sincosf(f, &sn, &cs);
  return float2{fmaf(-d, sn, cs) * scale, fmaf(d, cs, sn) * scale};
}

// 16-byte rows of head sizes 64, 128 and 256: a workgroup takes `per` tokens, whose (cos, sin) pairs
// go into LDS once for all heads; a head is HD / 2 / N lanes of two 16-byte vectors each, chosen so that a
// pair's two values are one lane's, and the next head's loads are out before this one's math.
// Bound by HBM: 16384 tokens of 28 / 4 heads of 128 with the store, bf16: 51.6 us,
// 5.9 TB/s (a large copy 6.5).
constexpr int kRotMaxTokens = 8;

template <typename T, int HD, bool INTERLEAVED>
__global__ __launch_bounds__(kRotThreads) void rotary_vec_kernel(const RotaryArgs<T> a, const FastDiv heads_div, int per) {
  constexpr int N = Pack<T>::N, LPH = HD / 2 / N, kHeads = kRotThreads / LPH;
  static_assert(LPH >= 1 && LPH <= 32 && (LPH & (LPH - 1)) == 0, "lanes of a head");
  __shared__ float2 cs[kRotMaxTokens * HD / 2];
  const int half = a.rot / 2, heads = a.q_heads + a.kv_heads;
  const int64_t t0 = (int64_t)blockIdx.x * per;
  const int n = a.tokens - t0 < per ? (int)(a.tokens - t0) : per;
  const int sub = threadIdx.x % LPH, items = n * heads;
  // this lane's vectors of a head, and whether they turn
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
    int64_t t;
    int h, i;
    u32x4 x1, x2, v1, v2;
    int32_t slot;
  };
  const auto load = [&](int at) {
    Item it{};
    it.i = (int)heads_div.div((uint32_t)at);
    it.t = t0 + it.i;
    it.h = at - it.i * heads;
    it.slot = -1;
    const bool is_q = it.h < a.q_heads;
    const int hk = it.h - a.q_heads;
    const T* x = is_q ? a.q + it.t * a.q_stride + (int64_t)it.h * HD : a.k + it.t * a.k_stride + (int64_t)hk * HD;
    it.x1 = ld16_nt(x + d1);
    it.x2 = ld16_nt(x + d2);
    if (!is_q && a.kc) {
      it.slot = a.slots[it.t];
      const T* v = a.v + it.t * a.v_stride + (int64_t)hk * HD;
      it.v1 = ld16_nt(v + d1);
      it.v2 = ld16_nt(v + d2);
    }
    return it;
  };
  int at = threadIdx.x / LPH;
  Item it{};
  if (at < items) it = load(at);
  for (int i = threadIdx.x; i < n * half; i += kRotThreads) {
    const int tk = i / half;
    cs[i] = rotary_cs(a.positions[t0 + tk], a.inv_freq[i - tk * half], a.attn_scale);
  }
  __syncthreads();
  for (; at < items; at += kHeads) {
    Item next{};
    if (at + kHeads < items) next = load(at + kHeads);
    float x1[N], x2[N];
    Pack<T>::unpack(it.x1, x1);
    Pack<T>::unpack(it.x2, x2);
    const bool is_q = it.h < a.q_heads;
    const T* w = is_q ? a.qw : a.kw;
    if (w) {
      float ss = 0.0f;
#pragma unroll
      for (int j = 0; j < N; ++j) ss = fmaf(x1[j], x1[j], fmaf(x2[j], x2[j], ss));
      const float inv = 1.0f / sqrtf(group_sum<LPH>(ss) / (float)HD + a.eps);
      float w1[N], w2[N];
      Pack<T>::unpack(ld16(w + d1), w1);
      Pack<T>::unpack(ld16(w + d2), w2);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        x1[j] = x1[j] * inv * w1[j];
        x2[j] = x2[j] * inv * w2[j];
      }
    }
    const float2* c = cs + it.i * half;
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
    const u32x4 y1 = Pack<T>::pack(x1), y2 = Pack<T>::pack(x2);
    const int hk = it.h - a.q_heads;
    T* y = is_q ? a.q_out + it.t * a.q_out_stride + (int64_t)it.h * HD
                : a.k_out ? a.k_out + it.t * a.k_out_stride + (int64_t)hk * HD : nullptr;
    if (y) {
      st16_nt(y + d1, y1);
      st16_nt(y + d2, y2);
    }
    if (it.slot >= 0 && it.slot < a.cache_rows) {
      const int64_t row = ((int64_t)it.slot * a.kv_heads + hk) * HD;
      st16(a.kc + row + d1, y1);
      st16(a.kc + row + d2, y2);
      st16(a.vc + row + d1, it.v1);
      st16(a.vc + row + d2, it.v2);
    }
    it = next;
  }
}

// Any head size, stride and alignment: a wave per (token, head), heads q then k; lanes walk the
// pairs, then the dimensions that are not rotated.
template <typename T>
__global__ __launch_bounds__(kRotThreads) void rotary_any_kernel(const RotaryArgs<T> a) {
  const int heads = a.q_heads + a.kv_heads, lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * (kRotThreads / 64) + threadIdx.x / 64;
  if (item >= a.tokens * heads) return;  // wave-uniform
  const int64_t t = item / heads;
  const int h = (int)(item - t * heads);
  const bool is_q = h < a.q_heads;
  const int hk = h - a.q_heads;
  const T* x = is_q ? a.q + t * a.q_stride + (int64_t)h * a.hd : a.k + t * a.k_stride + (int64_t)hk * a.hd;
  T* y = is_q ? a.q_out + t * a.q_out_stride + (int64_t)h * a.hd
              : a.k_out ? a.k_out + t * a.k_out_stride + (int64_t)hk * a.hd : nullptr;
  T* kc = nullptr;
  if (!is_q && a.kc) {
    const int32_t slot = a.slots[t];
    if (slot >= 0 && slot < a.cache_rows) {
      const int64_t at = ((int64_t)slot * a.kv_heads + hk) * a.hd;
      kc = a.kc + at;
      const T* v = a.v + t * a.v_stride + (int64_t)hk * a.hd;
      for (int d = lane; d < a.hd; d += 64) a.vc[at + d] = v[d];
    }
  }
  const T* w = is_q ? a.qw : a.kw;
  float inv = 1.0f;
  if (w) {
    float ss = 0.0f;
    for (int d = lane; d < a.hd; d += 64) {
      const float f = to_f32(x[d]);
      ss = fmaf(f, f, ss);
    }
    inv = 1.0f / sqrtf(wave_sum(ss) / (float)a.hd + a.eps);
  }
  const auto at = [&](int d) { return w ? to_f32(x[d]) * inv * to_f32(w[d]) : to_f32(x[d]); };
  const auto put = [&](int d, float f) {
    const T r = from_f32<T>(f);
    if (y) y[d] = r;
    if (kc) kc[d] = r;
  };
  const int64_t position = a.positions[t];
  for (int i = lane; i < a.rot / 2; i += 64) {
    const int da = a.interleaved ? 2 * i : i, db = a.interleaved ? 2 * i + 1 : i + a.rot / 2;
    const float2 cs = rotary_cs(position, a.inv_freq[i], a.attn_scale);
    const float x1 = at(da), x2 = at(db);
    put(da, x1 * cs.x - x2 * cs.y);
    put(db, x2 * cs.x + x1 * cs.y);
  }
  for (int d = a.rot + lane; d < a.hd; d += 64) put(d, at(d));
}

template <typename T, int HD>
void launch_rotary_vec(const RotaryArgs<T>& a, hipStream_t st) {
  constexpr int LPH = HD / 2 / Pack<T>::N;
  const int heads = a.q_heads + a.kv_heads;
  // tokens of a workgroup: enough heads for its threads, and a few passes of them where there are many tokens
  const int fill = (kRotThreads + heads * LPH - 1) / (heads * LPH);
  const int per = (int)std::min<int64_t>(kRotMaxTokens, std::max<int64_t>(fill, std::min<int64_t>(4, a.tokens / 2048)));
  const dim3 grid((unsigned)((a.tokens + per - 1) / per));
  const FastDiv div((uint32_t)heads);
  if (a.interleaved) rotary_vec_kernel<T, HD, true><<<grid, kRotThreads, 0, st>>>(a, div, per);
  else rotary_vec_kernel<T, HD, false><<<grid, kRotThreads, 0, st>>>(a, div, per);
}

template <typename T>
int rotary_dispatch(const RotaryArgs<T>& a, hipStream_t st) {
  constexpr int N = Pack<T>::N;
  const auto rows16 = [](const void* p, int64_t stride) { return !p || (aligned16(p) && stride % N == 0); };
  const bool vec = (a.interleaved ? a.rot : a.rot / 2) % N == 0 && rows16(a.q, a.q_stride) &&
                   rows16(a.q_out, a.q_out_stride) && rows16(a.k, a.k_stride) && rows16(a.k_out, a.k_out_stride) &&
                   rows16(a.v, a.v_stride) && rows16(a.kc, 0) && rows16(a.vc, 0) && rows16(a.qw, 0) && rows16(a.kw, 0);
  if (vec && a.hd == 64) launch_rotary_vec<T, 64>(a, st);
  else if (vec && a.hd == 128) launch_rotary_vec<T, 128>(a, st);
  else if (vec && a.hd == 256) launch_rotary_vec<T, 256>(a, st);
  else {
    const int64_t items = a.tokens * (a.q_heads + a.kv_heads), waves = kRotThreads / 64;
    rotary_any_kernel<T><<<dim3((unsigned)((items + waves - 1) / waves)), kRotThreads, 0, st>>>(a);
  }
  return launch_status("rotary");
}

}  // namespace nvf

using namespace nvf;

extern "C" {

int nvf_rotary(const void* q, void* q_out, const void* k, void* k_out, const void* v, const int64_t* positions,
               const double* inv_freq, int interleaved, int rotary_dim, float attn_scale, const void* q_w,
               const void* k_w, float eps, int64_t tokens, int q_heads, int kv_heads, int head_dim, int64_t q_stride,
               int64_t q_out_stride, int64_t k_stride, int64_t k_out_stride, int64_t v_stride, void* k_cache,
               void* v_cache, const int32_t* slot_mapping, int64_t cache_rows, int dtype, void* stream) {
  const char* who = "nvf_rotary";
  if (!dtype_ok(dtype)) return fail(NVF_ERR_INVALID, "%s: bad dtype %d", who, dtype);
  if (tokens < 0 || q_heads <= 0 || kv_heads < 0 || head_dim <= 0 || head_dim > 2 * kRotMaxPairs || cache_rows < 0)
    return fail(NVF_ERR_INVALID, "%s: bad shape tokens=%lld q_heads=%d kv_heads=%d head_dim=%d", who,
                (long long)tokens, q_heads, kv_heads, head_dim);
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2)
    return fail(NVF_ERR_INVALID, "%s: rotary_dim=%d is not an even part of head_dim=%d", who, rotary_dim, head_dim);
  const bool store = k_cache != nullptr;
  const int64_t qn = (int64_t)q_heads * head_dim, kn = (int64_t)kv_heads * head_dim;
  if (store && (!v_cache || !v || !slot_mapping || kv_heads == 0))
    return fail(NVF_ERR_INVALID, "%s: the store needs v, both caches and slot_mapping", who);
  if (q_stride < qn || q_out_stride < qn || (kv_heads > 0 && k_stride < kn) || (k_out && k_out_stride < kn) ||
      (store && v_stride < kn))
    return fail(NVF_ERR_INVALID, "%s: a stride is shorter than its row", who);
  if ((q_w == nullptr) != (k_w == nullptr)) return fail(NVF_ERR_INVALID, "%s: q_w and k_w go together", who);
  if (tokens == 0) return NVF_OK;
  if (!q || !q_out || !positions || (rotary_dim > 0 && !inv_freq) || (kv_heads > 0 && (!k || (!k_out && !store))))
    return fail(NVF_ERR_INVALID, "%s: NULL pointer", who);
  if (tokens * (q_heads + kv_heads) > INT32_MAX) return fail(NVF_ERR_INVALID, "%s: too many heads", who);
  const int e = dtype_bytes(dtype);
  // An output may be its own input and lie in other columns of the same packed rows, but not otherwise
  // over an input or the other output.
  struct Rows {
    const char* name;
    const void* p;
    int64_t stride, n;
  };
  const Rows in[] = {{"q", q, q_stride, qn}, {"k", k, k_stride, kn}, {"v", store ? v : nullptr, v_stride, kn}};
  const Rows out[] = {{"q_out", q_out, q_out_stride, qn}, {"k_out", k_out, k_out_stride, kn}};
  const auto clash = [&](const Rows& x, const Rows& y) {
    if (!x.p || !y.p || !bytes_overlap(x.p, ((tokens - 1) * x.stride + x.n) * e, y.p, ((tokens - 1) * y.stride + y.n) * e))
      return false;
    const int64_t d = static_cast<const char*>(y.p) - static_cast<const char*>(x.p);
    if (x.stride != y.stride || d % e) return true;
    const int64_t column = ((d / e) % x.stride + x.stride) % x.stride;  // of y's rows, seen from x's
    return column < x.n || column > x.stride - y.n;
  };
  for (int o = 0; o < 2; ++o)
    for (int i = 0; i < 3; ++i)
      if (clash(out[o], in[i]) && !(i == o && out[o].p == in[i].p && out[o].stride == in[i].stride))
        return fail(NVF_ERR_INVALID, "%s: %s overlaps %s", who, out[o].name, in[i].name);
  if (clash(out[0], out[1])) return fail(NVF_ERR_INVALID, "%s: q_out overlaps k_out", who);
  int rc = NVF_OK;
  NVF_DISPATCH_DTYPE(dtype, T, {
    RotaryArgs<T> a{};
    a.q = static_cast<const T*>(q);
    a.q_out = static_cast<T*>(q_out);
    a.k = static_cast<const T*>(k);
    a.k_out = static_cast<T*>(k_out);
    a.v = static_cast<const T*>(v);
    a.kc = static_cast<T*>(k_cache);
    a.vc = static_cast<T*>(v_cache);
    a.positions = positions;
    a.inv_freq = inv_freq;
    a.qw = static_cast<const T*>(q_w);
    a.kw = static_cast<const T*>(k_w);
    a.slots = slot_mapping;
    a.tokens = tokens;
    a.cache_rows = cache_rows;
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
    rc = rotary_dispatch<T>(a, as_stream(stream));
  });
  return rc;
}

// Host: the frequencies theta^(-2 i / rotary_dim), scaled for a longer context.
int nvf_rotary_inv_freq(double theta, int rotary_dim, int scaling, double factor, double low, double high,
                        double original_len, double* inv_freq, float* attn_scale) {
  const char* who = "nvf_rotary_inv_freq";
  if (rotary_dim <= 0 || rotary_dim % 2 || !(theta > 0.0) || !inv_freq || !attn_scale)
    return fail(NVF_ERR_INVALID, "%s: bad arguments", who);
  if (scaling < NVF_ROPE_PLAIN || scaling > NVF_ROPE_BANDS) return fail(NVF_ERR_INVALID, "%s: bad scaling %d", who, scaling);
  if (scaling != NVF_ROPE_PLAIN && !(factor >= 1.0)) return fail(NVF_ERR_INVALID, "%s: factor must be >= 1", who);
  if (scaling == NVF_ROPE_RAMP && !(theta > 1.0)) return fail(NVF_ERR_INVALID, "%s: theta must exceed 1", who);
  if (scaling >= NVF_ROPE_RAMP && (!(low > 0.0) || !(high > low) || !(original_len > 0.0)))
    return fail(NVF_ERR_INVALID, "%s: needs 0 < low < high and original_len > 0", who);
  const double two_pi = 6.283185307179586;
  // RAMP: the pair index at which a frequency turns `turns` times in original_len positions
  const auto pair_of = [&](double turns) {
    return rotary_dim * log(original_len / (turns * two_pi)) / (2.0 * log(theta));
  };
  const double first = scaling == NVF_ROPE_RAMP ? fmax(floor(pair_of(high)), 0.0) : 0.0;
  const double last = scaling == NVF_ROPE_RAMP ? fmin(ceil(pair_of(low)), rotary_dim - 1.0) : 0.0;
  for (int i = 0; i < rotary_dim / 2; ++i) {
    const double f = pow(theta, -2.0 * i / rotary_dim);
    double keep = 1.0;  // the share of the unscaled frequency
    if (scaling == NVF_ROPE_LINEAR) keep = 0.0;
    if (scaling == NVF_ROPE_RAMP) keep = 1.0 - fmin(fmax((i - first) / fmax(last - first, 1e-3), 0.0), 1.0);
    if (scaling == NVF_ROPE_BANDS) {
      const double turns = original_len * f / two_pi;
      keep = fmin(fmax((turns - low) / (high - low), 0.0), 1.0);
    }
    inv_freq[i] = f * keep + f / (scaling == NVF_ROPE_PLAIN ? 1.0 : factor) * (1.0 - keep);
  }
  *attn_scale = scaling == NVF_ROPE_RAMP ? (float)(0.1 * log(factor) + 1.0) : 1.0f;
  return NVF_OK;
}

}  // extern "C"
