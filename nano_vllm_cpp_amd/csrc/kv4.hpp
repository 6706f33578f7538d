// The 4-bit KV cache's rows.
//
// A row is one token: kv_heads x head_dim / 2 code bytes (dimension 2 b of a head in the low half of
// its byte b, 2 b + 1 in the high one), then kv_heads x head_dim / 32 words of 16 bits, then zeros to
// a multiple of 16 bytes.  Rows of a page lie side by side as those of other caches do, so pages are
// copied, forked and moved by the same calls.
//
// A word holds the 32 dimensions' scale and zero point: its upper 12 bits are those of an fp16 scale d
// (seven significant bits), the lower four z.  Code n stands for d (n - z): seven bits times four, so
// fp16 holds every value exactly and the 16-bit matrix cores read the cache without a rounding.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "nvf_device.hpp"

namespace nvf {

constexpr int kKv4Group = 32;          // dimensions of a scale
constexpr double kKv4MostScale = 4352.0;  // the largest scale of seven bits whose 15 steps fp16 holds
constexpr uint32_t kKv4NotANumber = 0x7E00;  // the word of a group that is no number: its values are NaN

inline int64_t kv4_row_bytes(int64_t kv_heads, int64_t head_dim) {
  return (kv_heads * (head_dim / 2 + head_dim / 16) + 15) / 16 * 16;
}
inline bool kv4_head_dim_ok(int head_dim) { return head_dim > 0 && head_dim <= 256 && head_dim % kKv4Group == 0; }

__device__ __forceinline__ float kv4_scale(uint32_t word) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)(word & 0xFFF0u));
}
__device__ __forceinline__ float kv4_value(uint32_t word, uint32_t code) {
  return kv4_scale(word) * (float)((int)code - (int)(word & 15u));
}

// A group's scale and zero point, from its least value or 0 and its largest or 0, in 64 bits: d is the
// least scale of seven significant bits (below 2^-14 the least multiple of 2^-20) that is not below (high -
// low) / 15, so that rounding codes to whole steps costs at most half a step, and z the whole step at -low.
struct Kv4Scale {
  double d, z;
  uint32_t word;
  __device__ __forceinline__ double inverse() const { return d > 0.0 ? 1.0 / d : 0.0; }  // (0: codes are z = 0)
};
__device__ __forceinline__ Kv4Scale kv4_scale_of(double low, double high) {
  const double need = (high - low) / 15.0;
  constexpr uint64_t kBelow = (1ull << 46) - 1;  // of a double's 52 fraction bits, those past the sixth
  const uint64_t up = (__builtin_bit_cast(uint64_t, need) + kBelow) & ~kBelow;
  double d = need >= 0x1p-14 ? __builtin_bit_cast(double, up) : ceil(need * 0x1p20) * 0x1p-20;
  d = fmin(d, kKv4MostScale);  // larger values saturate
  const double z = d > 0.0 ? fmin(rint(-low / d), 15.0) : 0.0;
  const uint16_t bits = __builtin_bit_cast(uint16_t, (_Float16)(float)d);
  return {d, z, (uint32_t)bits | (uint32_t)z};
}
// rint(x / d) + z within 0 .. 15.  x times the reciprocal, corrected by what is left of x, is the rounded quotient:
// exact where the quotient is a number of F's, so ties are ties.  (F fp32 for x of 16 bits: their quotients by a
// scale of seven bits lie 2^-13 off a tie or on it.)
template <typename F>
__device__ __forceinline__ uint32_t kv4_code(F x, F d, F z, F inv) {
  const F q = x * inv, left = __builtin_elementwise_fma(-q, d, x);
  const F n = __builtin_elementwise_rint(__builtin_elementwise_fma(left, inv, q)) + z;
  return (uint32_t)__builtin_elementwise_min(__builtin_elementwise_max(n, (F)0), (F)15);
}

}  // namespace nvf
