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

// (cos, sin) of position * freq, times the scale
__device__ __forceinline__ float2 rotary_cs(int64_t position, double freq, float scale) {
  const double t = (double)position * freq;
  const double n = rint(t * 0.15915494309189535);                             // 1 / (2 pi)
  const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, t));  // 2 pi in two parts
  const float x = (float)r;
  return float2{cosf(x) * scale, sinf(x) * scale};
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

template <typename T>
int rotary_dispatch(const RotaryArgs<T>& a, hipStream_t st) {
  const int64_t items = a.tokens * (a.q_heads + a.kv_heads), waves = kRotThreads / 64;
  rotary_any_kernel<T><<<dim3((unsigned)((items + waves - 1) / waves)), kRotThreads, 0, st>>>(a);
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
