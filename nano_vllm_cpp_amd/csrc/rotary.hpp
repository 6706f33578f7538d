// What the rotary entry points share: the angles, and the checks of a call.
#pragma once

#include <math.h>

#include "nvf_device.hpp"
#include "nvf_host.hpp"

namespace nvf {

constexpr int kRotMaxPairs = 128;  // of a head: head_dim <= 256

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

// (cos, sin) of position * freq, times the scale, in 64 bits: the angle less whole quarter turns (pi / 2 in two parts),
// and the series of both over [-pi/4, pi/4], whose next terms are below 2^-60.
struct Turn64 {
  double c, s;
};
__device__ __forceinline__ Turn64 rotary_cs64(int64_t position, double freq, double scale) {
  const double t = (double)position * freq;
  const double n = rint(t * 0.6366197723675814);  // 2 / pi
  const double r = fma(-n, 6.123233995736766e-17, fma(-n, 1.5707963267948966, t)), x = r * r;
  // 1 / (2 k + 1)! and 1 / (2 k)!, alternating
  double sn = fma(x, 2.8114572543455206e-15, -7.647163731819816e-13);
  sn = fma(x, sn, 1.6059043836821613e-10);
  sn = fma(x, sn, -2.505210838544172e-08);
  sn = fma(x, sn, 2.7557319223985893e-06);
  sn = fma(x, sn, -1.984126984126984e-04);
  sn = fma(x, sn, 8.333333333333333e-03);
  sn = fma(x, sn, -0.16666666666666666);
  sn = fma(r * x, sn, r);
  double cs = fma(x, -1.5619206968586225e-16, 4.779477332387385e-14);
  cs = fma(x, cs, -1.1470745597729725e-11);
  cs = fma(x, cs, 2.08767569878681e-09);
  cs = fma(x, cs, -2.755731922398589e-07);
  cs = fma(x, cs, 2.48015873015873e-05);
  cs = fma(x, cs, -1.388888888888889e-03);
  cs = fma(x, cs, 4.1666666666666664e-02);
  cs = fma(x, cs, -0.5);
  cs = fma(x, cs, 1.0);
  const int quarter = (int)(n - 4.0 * floor(n * 0.25));
  const double c = quarter & 1 ? sn : cs, s = quarter & 1 ? cs : sn;
  return {(quarter == 1 || quarter == 2 ? -c : c) * scale, (quarter >= 2 ? -s : s) * scale};
}

// The checks of a rotation with or without a store; NVF_OK with tokens > 0 means that a launch may follow.
inline int check_rotary(const char* who, const void* q, const void* q_out, const void* k, const void* k_out,
                        const void* v, const int64_t* positions, const double* inv_freq, int rotary_dim,
                        const void* q_w, const void* k_w, int64_t tokens, int q_heads, int kv_heads, int head_dim,
                        int64_t q_stride, int64_t q_out_stride, int64_t k_stride, int64_t k_out_stride,
                        int64_t v_stride, bool store, const void* v_cache, const int32_t* slot_mapping,
                        int64_t cache_rows, int dtype) {
  if (!dtype_ok(dtype)) return fail(NVF_ERR_INVALID, "%s: bad dtype %d", who, dtype);
  if (tokens < 0 || q_heads <= 0 || kv_heads < 0 || head_dim <= 0 || head_dim > 2 * kRotMaxPairs || cache_rows < 0)
    return fail(NVF_ERR_INVALID, "%s: bad shape tokens=%lld q_heads=%d kv_heads=%d head_dim=%d", who,
                (long long)tokens, q_heads, kv_heads, head_dim);
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2)
    return fail(NVF_ERR_INVALID, "%s: rotary_dim=%d is not an even part of head_dim=%d", who, rotary_dim, head_dim);
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
  return NVF_OK;
}

}  // namespace nvf
